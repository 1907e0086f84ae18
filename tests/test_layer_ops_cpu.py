"""What the norm, routing and 4-bit entry points refuse, before anything reaches a GPU."""
import ctypes
import os
import re

import pytest
import torch

from tests.conftest import ROOT

A16, ODD = 4096, 4100                 # never dereferenced: an aligned and an unaligned address


@pytest.fixture(scope="module")
def lib():
    from tirx_harness_b200 import _lib, build
    build.build_library()
    return _lib


def _refused(lib, fn, args, *words):
    rc = getattr(lib.lib(), fn)(ctypes.byref(args), None)
    message = lib.lib().moe_last_error().decode()
    assert rc == -1, (rc, message)
    for w in words:
        assert w in message, message


def _norm(lib, **kw):
    base = dict(x=A16, x_stride=256, residual=A16, residual_stride=256, weight=A16, q=A16, scales=A16, ss_row=2, ss_blk=1, h=A16, y=A16,
                rstd=A16, T=4, H=256, dtype=0, w_dtype=0, pow2=0, eps=1e-6)
    return lib.NormArgs(**(base | kw))


@pytest.mark.parametrize("kw,word", [
    (dict(T=-1), "T=-1"), (dict(H=0), "H=0"), (dict(H=12), "H=12"), (dict(H=16392), "H=16392"), (dict(dtype=7), "dtype"), (dict(dtype=0, w_dtype=2), "dtype"),
    (dict(x=None), "x"), (dict(x=ODD), "x"), (dict(x_stride=248), "x"), (dict(x_stride=260), "x"), (dict(residual_stride=128), "residual"),
    (dict(residual=ODD), "residual"), (dict(h=None), "h"), (dict(weight=None), "weight"), (dict(q=None), "q"), (dict(scales=None), "scales"),
    (dict(rstd=None), "rstd"), (dict(y=ODD), "y"), (dict(q=ODD), "q")])
def test_norm_refuses(lib, kw, word):
    _refused(lib, "moe_rms_norm_quant", _norm(lib, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(T=-1), "T=-1"), (dict(H=20), "H=20"), (dict(dtype=1, w_dtype=0), "dtype"), (dict(dw=None), "dw"), (dict(dy=None), "dy"), (dict(h=ODD), "h"),
    (dict(dh=A16, dh_stride=8), "dh"), (dict(dx=None), "dx"), (dict(rstd=None), "rstd"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=100), "workspace")])
def test_norm_gradient_refuses(lib, kw, word):
    base = dict(dy=A16, dy_stride=256, h=A16, h_stride=256, weight=A16, rstd=A16, dh=None, dh_stride=0, dx=A16, dw=A16, T=4, H=256, dtype=0,
                w_dtype=0, workspace=A16, workspace_bytes=1 << 20)
    _refused(lib, "moe_rms_norm_backward", lib.NormGradArgs(**(base | kw)), word)


ROUTE = dict(logits=A16, stride=256, bias=A16, ids=A16, weights=A16, T=4, E=256, top_k=8, n_group=8, topk_group=4, dtype=1, bias_dtype=1, score=1,
             group_score=1, renormalize=1, scale=1.0)


@pytest.mark.parametrize("kw,word", [
    (dict(T=-2), "T=-2"), (dict(E=0), "E=0"), (dict(E=1025, stride=1025), "E=1025"), (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"), (dict(stride=255), "stride"),
    (dict(dtype=5), "dtype"), (dict(score=2), "score"), (dict(n_group=0), "n_group"), (dict(n_group=7), "n_group"), (dict(n_group=64), "n_group"),
    (dict(topk_group=9), "topk_group"), (dict(topk_group=0), "topk_group"), (dict(n_group=32, topk_group=1, top_k=9), "top_k"), (dict(group_score=3), "group_score"),
    (dict(bias_dtype=2), "bias_dtype"), (dict(logits=None), "logits"), (dict(ids=None), "ids")])
def test_route_refuses(lib, kw, word):
    _refused(lib, "moe_route", lib.RouteArgs(**(ROUTE | kw)), word)


@pytest.mark.parametrize("kw,word", [(dict(E=2000, stride=2000), "E=2000"), (dict(top_k=40), "top_k"), (dict(grad_weights=None), "grad_weights"), (dict(dlogits=None), "dlogits")])
def test_route_gradient_refuses(lib, kw, word):
    base = dict(grad_weights=A16, logits=A16, stride=64, ids=A16, dlogits=A16, T=4, E=64, top_k=8, dtype=1, score=0, renormalize=1, scale=1.0)
    _refused(lib, "moe_route_backward", lib.RouteGradArgs(**(base | kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(groups=0), "groups"), (dict(rows=-1), "rows"), (dict(K=192), "K=192"), (dict(K=0), "K=0"), (dict(format=2), "format"), (dict(dtype=9), "dtype"),
    (dict(src_rows=5), "src_rows"), (dict(src_pair=A16, groups=2), "src_pair"), (dict(src_pair=A16, top_k=0), "top_k"), (dict(format=1, factor=A16), "factor"),
    (dict(x=None), "x"), (dict(x=ODD), "x"), (dict(x_stride=100), "x"), (dict(silu_mul=1), "x"), (dict(q=None), "q"), (dict(scales=ODD), "scales")])
def test_quant_fp4_refuses(lib, kw, word):
    base = dict(x=A16, x_stride=256, factor=None, factor_stride=0, src_pair=None, q=A16, scales=A16, groups=1, rows=4, src_rows=4, K=256, top_k=1, dtype=0,
                format=0, silu_mul=0, gate_first=1)
    _refused(lib, "moe_quant_fp4", lib.Fp4QuantArgs(**(base | kw)), word)


def test_quant_fp4_workspace(lib):
    need = lib.lib().moe_quant_fp4_workspace_bytes
    assert need(8192, 4096, 2048, 0) == 4096 * (1024 + 8 * 16) and need(8192, 4096, 2048, 1) == 4096 * (1024 + 8 * 8)
    assert need(8192, 4097, 2048, 0) == 0 and need(4095, 1000, 2048, 0) == 0         # too few rows for one of x, too few values
    for bad in ((-1, 1, 256, 0), (8192, 0, 2048, 0), (8192, 4096, 2000, 0), (8192, 4096, 2048, 2)):
        assert need(*bad) == 0
    base = dict(x=A16, x_stride=2048, src_pair=A16, q=A16, scales=A16, groups=1, rows=8192, src_rows=4096, K=2048, top_k=2, gate_first=1)
    full = need(8192, 4096, 2048, 0)
    for kw in (dict(workspace=A16, workspace_bytes=full - 1), dict(workspace=ODD, workspace_bytes=full)):
        _refused(lib, "moe_quant_fp4", lib.Fp4QuantArgs(**(base | kw)), "workspace")


@pytest.mark.parametrize("fn", ["moe_gg_fp4_contiguous", "moe_gg_fp4_masked"])
@pytest.mark.parametrize("kw,word", [
    (dict(G=0), "G"), (dict(M=-1), "M"), (dict(N=20), "N=20"), (dict(K=64), "K=64"), (dict(format=5), "format"), (dict(d_dtype=2), "d_dtype"), (dict(ldd=48), "ldd"),
    (dict(ldd=65), "ldd"), (dict(alpha=A16, alpha_stride=2), "alpha_stride"), (dict(a=None), "a"), (dict(sfb=None), "sfb"), (dict(d=ODD), "16-byte"),
    (dict(sfa=ODD), "16-byte"), (dict(G=1 << 20, N=1 << 12, ldd=1 << 12), "")])
def test_product_refuses(lib, fn, kw, word):
    base = dict(a=A16, sfa=A16, b=A16, sfb=A16, alpha=None, alpha_stride=0, layout=A16, rows_used=None, d=A16, ldd=64, G=2, M=4, N=64, K=256, format=0, d_dtype=0)
    _refused(lib, fn, lib.GGFp4Args(**(base | kw)), word)


def test_row_counts_at_the_end_of_32_bits_are_refused(lib):
    """Rounded up to whole blocks they would pass 2^31."""
    top = (1 << 31) - 1
    for T in (top, top - 126):
        _refused(lib, "moe_route", lib.RouteArgs(**(ROUTE | dict(T=T))), "T=")
        _refused(lib, "moe_route_backward", lib.RouteGradArgs(grad_weights=A16, logits=A16, stride=64, ids=A16, dlogits=A16, T=T, E=64, top_k=8, dtype=1), "T=")
        quant = dict(x=A16, x_stride=256, src_pair=A16, q=A16, scales=A16, groups=1, rows=T, src_rows=4, K=128, top_k=1, gate_first=1)
        _refused(lib, "moe_quant_fp4", lib.Fp4QuantArgs(**quant), "rows=")
        product = dict(a=A16, sfa=A16, b=A16, sfb=A16, layout=A16, d=A16, ldd=64, G=1, M=T, N=64, K=128)
        for fn in ("moe_gg_fp4_contiguous", "moe_gg_fp4_masked"):
            _refused(lib, fn, lib.GGFp4Args(**product), "scales")
            _refused(lib, fn, lib.GGFp4Args(**(product | dict(M=4, N=top - 7, ldd=top - 7))), "scales")


def test_unpack_refuses(lib):
    f = lib.lib().moe_unpack_fp4
    p = ctypes.c_void_p
    for q, out, n in ((A16, A16, 12), (A16, A16, -8), (None, A16, 8), (A16, ODD, 8)):
        assert f(p(q), p(out), ctypes.c_int64(n), None) == -1


def test_nothing_to_do_is_no_error(lib):
    L = lib.lib()
    assert L.moe_rms_norm_quant(ctypes.byref(_norm(lib, T=0, x=None)), None) == 0
    assert L.moe_route(ctypes.byref(lib.RouteArgs(**(ROUTE | dict(T=0, logits=None)))), None) == 0
    assert L.moe_unpack_fp4(None, None, ctypes.c_int64(0), None) == 0
    for fn in ("moe_rms_norm_quant", "moe_route", "moe_route_backward", "moe_quant_fp4", "moe_gg_fp4_contiguous", "moe_gg_fp4_masked", "moe_rms_norm_backward"):
        assert getattr(L, fn)(None, None) == -1


def test_tensors_on_the_host_are_refused():
    from tirx_harness_b200 import grouped_gemm, moe_ops
    x, w = torch.zeros((4, 256)), torch.ones(256)
    for call in (lambda: moe_ops.rms_norm_quant(x, w), lambda: moe_ops.rms_norm_backward(x, x, w, torch.ones(4)), lambda: moe_ops.route(x, 2),
                 lambda: moe_ops.route_backward(torch.zeros(4, 2), x, torch.zeros((4, 2), dtype=torch.int32)), lambda: moe_ops.quant_fp4(x),
                 lambda: moe_ops.unpack_fp4(torch.zeros(16, dtype=torch.uint8)),
                 lambda: grouped_gemm.bind_masked_fp4(torch.zeros((1, 4, 128), dtype=torch.uint8), x, torch.zeros((1, 8, 128), dtype=torch.uint8), x, x, x)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        moe_ops.route(x.long(), 2)


@pytest.mark.parametrize("at,value,error,word", [
    ("T", 1 << 31, ValueError, "T=2147483648"), ("stride", 1 << 63, ValueError, "stride="), ("n_group", 2.0, TypeError, "n_group"),
    ("topk_group", "2", TypeError, "topk_group"), ("scale", None, TypeError, "scale"), ("scale", 10**400, ValueError, "scale=")])
def test_values_that_do_not_fit_are_refused_by_name(lib, at, value, error, word):
    """Before any CUDA call, and as the other checks of arguments refuse."""
    from tirx_harness_b200 import moe_ops
    block = dict(logits=A16, stride=64, bias=0, ids=A16, weights=A16, T=4, E=64, top_k=2, n_group=1, topk_group=1, dtype=0, bias_dtype=0,
                 score=0, group_score=0, renormalize=1, scale=1.0)
    assert list(block) == [f[0] for f in lib.RouteArgs._fields_]
    block[at] = value
    with pytest.raises(error, match=word):
        moe_ops._launch(lib.ROUTE, torch.device("cuda", 0), *block.values())


def test_scale_tile_shapes():
    from tirx_harness_b200 import moe_ops
    assert moe_ops.fp4_scale_shape(1, 128, "nvfp4") == (1, 4, 512)
    assert moe_ops.fp4_scale_shape(129, 384, "mxfp4") == (2, 4, 512)
    assert moe_ops.fp4_scale_shape(0, 256, "mxfp4") == (0, 2, 512)
    with pytest.raises(ValueError):
        moe_ops.fp4_scale_shape(1, 128, "fp4")


def test_struct_layouts_match_header_field_order(lib):
    text = open(os.path.join(ROOT, "include", "b200moe.h")).read()
    for cname, pystruct in (("moe_norm_args", lib.NormArgs), ("moe_norm_grad_args", lib.NormGradArgs), ("moe_route_args", lib.RouteArgs),
                            ("moe_route_grad_args", lib.RouteGradArgs), ("moe_fp4_quant_args", lib.Fp4QuantArgs), ("moe_gg_fp4_args", lib.GGFp4Args)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            names = decl.split(None, 1)[1] if not decl.startswith("const") else decl.split(None, 2)[2]
            fields += [n.strip().lstrip("*").strip() for n in names.split(",")]
        assert fields == [f[0] for f in pystruct._fields_], cname
