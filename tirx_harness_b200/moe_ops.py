"""Host wrappers of the memory-bound stages around the grouped GEMMs (PyTorch tensors -> C ABI)."""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


def _stream(t: torch.Tensor):
    return _vp(torch.cuda.current_stream(t.device).cuda_stream)


def _scale_out(rows: int, nb: int, mn_major: bool, device):
    """Allocates a [rows, nb] scale tensor, physically [nb, rows] when mn_major."""
    if mn_major:
        return torch.empty((nb, rows), dtype=torch.float32, device=device).t()
    return torch.empty((rows, nb), dtype=torch.float32, device=device)


def quant_1x128(x: torch.Tensor, mn_major: bool = False, out=None):
    """bf16 [rows, cols] -> (e4m3 [rows, cols], f32 scales [rows, cols/128])."""
    assert x.dtype == torch.bfloat16 and x.is_cuda and x.is_contiguous() and x.dim() == 2
    rows, cols = x.shape
    q, s = out if out is not None else (torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=x.device),
                                        _scale_out(rows, cols // 128, mn_major, x.device))
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().moe_quant_1x128(_vp(x.data_ptr()), _vp(q.data_ptr()), _vp(s.data_ptr()),
                                              _i64(s.stride(0)), _i64(s.stride(1)), _i32(rows), _i32(cols), _stream(x)))
    return q, s


def silu_mul_requant(gate_up: torch.Tensor, gate_first: bool = True, layout=None, mn_major: bool = False, out=None):
    """bf16 [rows, 2I] -> (e4m3 [rows, I], f32 scales [rows, I/128]); rows with layout < 0 are skipped."""
    assert gate_up.dtype == torch.bfloat16 and gate_up.is_cuda and gate_up.is_contiguous()
    rows, two_i = gate_up.shape
    inter = two_i // 2
    q, s = out if out is not None else (torch.zeros((rows, inter), dtype=torch.float8_e4m3fn, device=gate_up.device),
                                        _scale_out(rows, inter // 128, mn_major, gate_up.device).zero_())
    with torch.cuda.device(gate_up.device):
        _lib.check(_lib.lib().moe_silu_mul_requant(
            _vp(gate_up.data_ptr()), _vp(q.data_ptr()), _vp(s.data_ptr()), _i64(s.stride(0)), _i64(s.stride(1)),
            _vp(layout.data_ptr()) if layout is not None else None, _i32(rows), _i32(inter),
            _i32(1 if gate_first else 0), _stream(gate_up)))
    return q, s


def route_topk(logits: torch.Tensor, top_k: int):
    """f32 [T, E] -> (ids int32 [T, top_k], weights f32 [T, top_k])."""
    assert logits.dtype == torch.float32 and logits.is_cuda and logits.is_contiguous()
    T, E = logits.shape
    ids = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        _lib.check(_lib.lib().moe_route_topk(_vp(logits.data_ptr()), _vp(ids.data_ptr()), _vp(w.data_ptr()),
                                             _i32(T), _i32(E), _i32(top_k), _stream(logits)))
    return ids, w


def route_deepseek(logits: torch.Tensor, bias: torch.Tensor, top_k: int = 8, n_group: int = 8, topk_group: int = 4,
                   routed_scaling_factor: float = 1.0):
    """DeepSeek-V3 no-aux routing: f32 [T, E], bias bf16/f32 [E] -> (ids int32 [T, top_k], weights f32 [T, top_k])."""
    assert logits.dtype == torch.float32 and logits.is_cuda and logits.is_contiguous()
    assert bias.dtype in (torch.bfloat16, torch.float32) and bias.is_contiguous()
    T, E = logits.shape
    ids = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        _lib.check(_lib.lib().moe_route_deepseek(_vp(logits.data_ptr()), _vp(bias.data_ptr()),
                                                 _i32(0 if bias.dtype == torch.bfloat16 else 1), _vp(ids.data_ptr()),
                                                 _vp(w.data_ptr()), _i32(T), _i32(E), _i32(n_group), _i32(topk_group),
                                                 _i32(top_k), ctypes.c_float(routed_scaling_factor), _stream(logits)))
    return ids, w


def plan_cap_rows(n_pairs: int, e_local: int, align: int) -> int:
    return (n_pairs + align - 1) // align * align + e_local * align


def permute_plan(ids: torch.Tensor, e_lo: int, e_local: int, align: int = 128, cap_rows: int | None = None):
    """ids int32 [T, top_k] (or flat) -> dict(counts, offsets, pos, src_pair, grouped_layout, cap_rows)."""
    assert ids.dtype == torch.int32 and ids.is_cuda and ids.is_contiguous()
    n = ids.numel()
    dev = ids.device
    cap = plan_cap_rows(n, e_local, align) if cap_rows is None else cap_rows
    counts = torch.empty(e_local, dtype=torch.int32, device=dev)
    offsets = torch.empty(e_local + 1, dtype=torch.int32, device=dev)
    pos = torch.empty(ids.shape, dtype=torch.int32, device=dev)
    src = torch.empty(cap, dtype=torch.int32, device=dev)
    gl = torch.empty(cap, dtype=torch.int32, device=dev)
    L = _lib.lib()
    ws_bytes = L.moe_permute_workspace_bytes(_i64(n), _i32(e_local))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.moe_permute_plan(_vp(ids.data_ptr()), _i64(n), _i32(e_lo), _i32(e_local), _i32(align), _i32(cap),
                                      _vp(counts.data_ptr()), _vp(offsets.data_ptr()), _vp(pos.data_ptr()),
                                      _vp(src.data_ptr()), _vp(gl.data_ptr()), _vp(ws.data_ptr()),
                                      ctypes.c_size_t(ws_bytes), _stream(ids)))
    return dict(counts=counts, offsets=offsets, pos=pos, src_pair=src, grouped_layout=gl, cap_rows=cap)


def permute(x_q: torch.Tensor, x_scale: torch.Tensor, src_pair: torch.Tensor, top_k: int, mn_major: bool = True,
            out=None):
    """Gathers token rows into the grouped layout: -> (a e4m3 [rows, H], scales f32 [rows, H/128])."""
    T, H = x_q.shape
    rows = src_pair.numel()
    a, s = out if out is not None else (torch.zeros((rows, H), dtype=torch.float8_e4m3fn, device=x_q.device),
                                        _scale_out(rows, H // 128, mn_major, x_q.device).zero_())
    with torch.cuda.device(x_q.device):
        _lib.check(_lib.lib().moe_permute(_vp(x_q.data_ptr()), _vp(x_scale.data_ptr()), _i64(x_scale.stride(0)),
                                          _i64(x_scale.stride(1)), _vp(src_pair.data_ptr()), _i32(top_k),
                                          _vp(a.data_ptr()), _vp(s.data_ptr()), _i64(s.stride(0)), _i64(s.stride(1)),
                                          _i32(rows), _i32(H), _stream(x_q)))
    return a, s


def combine(y: torch.Tensor, pos: torch.Tensor, w: torch.Tensor, out=None):
    """y bf16 [rows, H], pos int32 [T, top_k], w f32 [T, top_k] -> bf16 [T, H]."""
    T, top_k = pos.shape
    H = y.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16, device=y.device)
    with torch.cuda.device(y.device):
        _lib.check(_lib.lib().moe_combine(_vp(y.data_ptr()), _vp(pos.data_ptr()), _vp(w.data_ptr()), _vp(out.data_ptr()),
                                          _i32(T), _i32(top_k), _i32(H), _stream(y)))
    return out


# ------------------------------------------------------------------ norm, routing and 4-bit operands
_DTYPE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}
FP4_BLOCK = {"nvfp4": 16, "mxfp4": 32}           # values under one scale
_FP4_FORMAT = {"nvfp4": _lib.FP4_NV, "mxfp4": _lib.FP4_MX}


def _p(t):
    return 0 if t is None else t.data_ptr()


def _check_float(t, name, dtypes=_DTYPE):
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


def _check_like(t, name, shape, dtype, device, contiguous=True):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _rows(t, name, step=8):
    """(rows, columns, elements between rows) of a 2-d tensor whose columns are next to one another; a single row's distance
    does not matter and is given as one that its columns and ``step`` allow."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {t.dim()}")
    (n, cols), (ld, unit) = t.shape, t.stride()
    if unit != 1 and cols > 1:
        raise ValueError(f"{name} must have unit column stride")
    return n, cols, ld if n > 1 else (cols + step - 1) // step * step


# the current stream of a device as an integer, without the object that torch.cuda.current_stream makes
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(entry, device, *values):
    """Calls an entry point on the current stream of the tensors' device, which need not be the current one."""
    try:
        block = entry.pack(*values)
    except (struct.error, OverflowError):
        raise entry.misfit(values) from None
    index = device.index
    if index == torch.cuda.current_device():
        entry(block, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            entry(block, _raw_stream(index))


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                   pow2: bool = False, mn_major: bool = False, want_y: bool = False):
    """Residual addition, root-mean-square norm and 1x128 quantisation in one pass.

    x, residual bf16/f16/f32 [T, H] (any row stride that is a multiple of 8), weight [H] of x's type or f32 ->
    dict(q e4m3 [T, H], scales f32 [T, ceil(H/128)], h, y, rstd f32 [T]) with h = round(x + residual) (x itself without a
    residual), y = h * rstd * weight (x's type; None unless ``want_y``) and q, scales its 1x128 quantisation as
    :func:`quant_1x128` does it, from y in fp32.  ``pow2`` rounds the scales up to powers of two, which the grouped GEMM
    applies inside the tensor core; ``mn_major`` stores them [H/128, T].  H % 8 == 0, H <= 16384.

    Autograd does not see the call: the results carry no gradient, :func:`rms_norm_backward` computes it."""
    _check_float(x, "x")
    T, H, ld = _rows(x, "x")
    dt, dev = x.dtype, x.device
    if weight.dtype != dt and weight.dtype != torch.float32:
        raise TypeError(f"weight must be {dt} or float32, got {weight.dtype}")
    _check_like(weight, "weight", (H,), weight.dtype, dev)
    ldr, h, y = 0, x, None
    if residual is not None:
        _check_like(residual, "residual", x.shape, dt, dev, contiguous=False)
        ldr = _rows(residual, "residual")[2]
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    if want_y:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
    nb = (H + 127) // 128
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    s = x.new_empty((nb, T) if mn_major else (T, nb), dtype=torch.float32)
    rstd = x.new_empty(T, dtype=torch.float32)
    _launch(_lib.NORM, dev, x.data_ptr(), ld, _p(residual), ldr, weight.data_ptr(), q.data_ptr(), s.data_ptr(),
            1 if mn_major else nb, T if mn_major else 1, h.data_ptr() if residual is not None else 0, _p(y), rstd.data_ptr(),
            T, H, _DTYPE[dt], _DTYPE[weight.dtype], 1 if pow2 else 0, eps)
    return dict(q=q, scales=s.t() if mn_major else s, h=h, y=y, rstd=rstd)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dh: torch.Tensor | None = None):
    """Gradient of :func:`rms_norm_quant`, the rounding to 8 bits passed through unchanged.

    dy = dL/dy and h [T, H] of one type, rstd from the forward call, dh (optional) the gradient that reaches h past the
    norm -> (dx [T, H], the gradient of x and of residual alike; dw f32 [H])."""
    _check_float(dy, "dy")
    T, H, ld = _rows(dy, "dy")
    dt, dev = dy.dtype, dy.device
    _check_like(h, "h", dy.shape, dt, dev, contiguous=False)
    if weight.dtype != dt and weight.dtype != torch.float32:
        raise TypeError(f"weight must be {dt} or float32, got {weight.dtype}")
    _check_like(weight, "weight", (H,), weight.dtype, dev)
    _check_like(rstd, "rstd", (T,), torch.float32, dev)
    ldd = 0
    if dh is not None:
        _check_like(dh, "dh", dy.shape, dt, dev, contiguous=False)
        ldd = _rows(dh, "dh")[2]
    dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
    dw = dy.new_empty(H, dtype=torch.float32)
    n = _lib.lib().moe_rms_norm_backward_workspace_bytes(_i32(T), _i32(H))
    ws = dy.new_empty(n, dtype=torch.uint8)
    _launch(_lib.NORM_GRAD, dev, dy.data_ptr(), ld, h.data_ptr(), _rows(h, "h")[2], weight.data_ptr(), rstd.data_ptr(), _p(dh), ldd,
            dx.data_ptr(), dw.data_ptr(), T, H, _DTYPE[dt], _DTYPE[weight.dtype], ws.data_ptr(), n)
    return dx, dw


_BIAS_DTYPE = (torch.bfloat16, torch.float32)
_SCORE = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}


def _choice(table, value, name):
    if value not in table:
        raise ValueError(f"{name} must be one of {', '.join(table)}, got {value!r}")
    return table[value]


def route(logits: torch.Tensor, top_k: int, score: str = "softmax", bias: torch.Tensor | None = None, n_group: int = 1,
          topk_group: int = 1, group_score: str = "top2", renormalize: bool = True, scale: float = 1.0):
    """Top-k routing: bf16/f16/f32 [T, E] -> (ids int32 [T, top_k], weights f32 [T, top_k]).

    p = softmax or sigmoid of the logits; the experts are chosen by p + bias (bf16/f32 [E]) as 64 bits order it (without a
    bias: in the logits' order), ties to the lowest index, and weighted by p (over its sum of the chosen with
    ``renormalize``) * scale.  With n_group > 1 only the
    topk_group best groups of E / n_group consecutive experts count; a group's score is its best p + bias ("max") or the
    sum of its two best ("top2").  A logit or bias of -inf or NaN switches its expert off (+inf counts as the largest
    number); where fewer than top_k experts are left the id is -1 and the weight 0, which :func:`permute_plan` drops.
    E <= 1024, top_k <= 32, n_group <= 32.

    It covers the rules of :func:`route_topk` and :func:`route_deepseek` and is faster than either at every size.  Autograd
    does not see the call: the weights carry no gradient, :func:`route_backward` computes it."""
    _check_float(logits, "logits")
    T, E, ld = _rows(logits, "logits", 1)
    if bias is not None:
        _check_float(bias, "bias", _BIAS_DTYPE)
        _check_like(bias, "bias", (E,), bias.dtype, logits.device)
    if not 0 < top_k <= min(32, E):
        raise ValueError(f"top_k must be in [1, min(32, E)], got {top_k}")
    ids = logits.new_empty((T, top_k), dtype=torch.int32)
    w = logits.new_empty((T, top_k), dtype=torch.float32)
    _launch(_lib.ROUTE, logits.device, logits.data_ptr(), ld, _p(bias), ids.data_ptr(), w.data_ptr(), T, E, top_k, n_group, topk_group,
            _DTYPE[logits.dtype], 0 if bias is None else _DTYPE[bias.dtype], _choice(_SCORE, score, "score"),
            _choice(_GROUP_SCORE, group_score, "group_score"), 1 if renormalize else 0, scale)
    return ids, w


def route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, score: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0):
    """Gradient of :func:`route`'s weights with respect to the logits, the choice held fixed: [T, E] of the logits' type."""
    _check_float(logits, "logits")
    T, E, ld = _rows(logits, "logits", 1)
    if ids.dim() != 2:
        raise ValueError("ids must be [T, top_k]")
    top_k = ids.shape[1]
    _check_like(ids, "ids", (T, top_k), torch.int32, logits.device)
    _check_like(grad_weights, "grad_weights", (T, top_k), torch.float32, logits.device)
    out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    _launch(_lib.ROUTE_GRAD, logits.device, grad_weights.data_ptr(), logits.data_ptr(), ld, ids.data_ptr(), out.data_ptr(), T, E, top_k,
            _DTYPE[logits.dtype], _choice(_SCORE, score, "score"), 1 if renormalize else 0, scale)
    return out


def fp4_scale_shape(rows: int, K: int, fmt: str = "nvfp4"):
    """Shape of the scale tiles of ``rows`` x K values: uint8 [ceil(rows/128), ceil(K/256) * (4 nvfp4, 2 mxfp4), 512];
    row r's bytes of a tile's four blocks are at (r % 32) * 16 + (r // 32 % 4) * 4."""
    return ((rows + 127) // 128, (K + 255) // 256 * (64 // _choice(FP4_BLOCK, fmt, "fmt")), 512)


def quant_fp4(x: torch.Tensor, fmt: str = "nvfp4", global_scale: torch.Tensor | None = None, act: str | None = None,
              gate_first: bool = True, src_pair: torch.Tensor | None = None, top_k: int = 1, out=None):
    """Quantises to 4-bit blocks: -> (codes uint8 [.., rows, K/2], scale tiles uint8 [.., *fp4_scale_shape(rows, K, fmt)]).

    x bf16/f16/f32 [rows, K] (row stride a multiple of 8) or, for operands of several groups, contiguous [G, rows, K].
      fmt          "nvfp4": one e4m3 scale per 16 values under ``global_scale`` (f32, one value or [G], positive and finite;
                   default 1): s = e4m3(min(amax / (6 g), 448)), value = code * s * g.  "mxfp4": a power of two per 32 values
      global_scale largest magnitude / (6 * 448) uses the scales' whole range.  With 1 a block whose largest magnitude is at
                   most 0.0059 (6 * 2^-10) becomes zero: too large a factor for most weights
      act          "silu_mul": x is [rows, 2K] and SiLU(gate) * up, in fp32, is quantised (gate = the first half, or the
                   second with gate_first=False)
      src_pair     int32 [rows]: row r is made from x[src_pair[r] // top_k], as :func:`permute` gathers; where it is negative
                   the row of ``out`` is left as it is.  From twice as many rows as x has on, all of x is quantised once and
                   its rows are copied, whatever share of the rows is negative
      out          (codes, scales) to write into; without it codes and scales of skipped rows are zero
    K % 128 == 0.  A block that holds an infinity or a NaN gets the scale NaN."""
    _check_float(x, "x")
    block = _choice(FP4_BLOCK, fmt, "fmt")
    if act not in (None, "silu_mul"):
        raise ValueError(f"act must be None or 'silu_mul', got {act!r}")
    if x.dim() == 3:
        if not x.is_contiguous():
            raise ValueError("a three-dimensional x must be contiguous")
        G, src_rows, cols = x.shape
        ld, lead = cols, (G,)
    else:
        (src_rows, cols, ld), G, lead = _rows(x, "x"), 1, ()
    if act is not None and cols % 2:
        raise ValueError("with act='silu_mul' x must be [rows, 2K]")
    K = cols // 2 if act is not None else cols
    if K == 0 or K % 128:
        raise ValueError(f"K={K} must be a positive multiple of 128")
    rows = src_rows
    if src_pair is not None:
        if G != 1 or x.dim() == 3:
            raise ValueError("src_pair needs a two-dimensional x")
        _check_like(src_pair, "src_pair", (src_pair.numel(),), torch.int32, x.device)
        if top_k < 1:
            raise ValueError("top_k must be positive")
        rows = src_pair.numel()
    gs = 0
    if global_scale is not None:
        if fmt != "nvfp4":
            raise ValueError("global_scale belongs to nvfp4")
        if global_scale.numel() not in (1, G):
            raise ValueError(f"global_scale must hold one value or {G}")
        _check_like(global_scale, "global_scale", global_scale.shape, torch.float32, x.device)
        gs = 1 if global_scale.numel() > 1 else 0
    q_shape, s_shape = (*lead, rows, K // 2), (*lead, *fp4_scale_shape(rows, K, fmt))
    if out is not None:
        q, s = out
        _check_like(q, "out[0]", q_shape, torch.uint8, x.device)
        _check_like(s, "out[1]", s_shape, torch.uint8, x.device)
    else:
        make = x.new_empty if src_pair is None else x.new_zeros
        q, s = make(q_shape, dtype=torch.uint8), make(s_shape, dtype=torch.uint8)
    if G == 0 or rows == 0:
        return q, s
    ws, n = None, 0
    if rows > src_rows and act is None:                      # gathered with several rows for one of x: it is quantised once
        n = _lib.lib().moe_quant_fp4_workspace_bytes(_i32(rows), _i32(src_rows), _i32(K), _i32(_FP4_FORMAT[fmt]))
        ws = x.new_empty(n, dtype=torch.uint8) if n else None
    _launch(_lib.FP4_QUANT, x.device, x.data_ptr(), ld, _p(global_scale), gs, _p(src_pair), q.data_ptr(), s.data_ptr(), G, rows, src_rows, K,
            top_k, _DTYPE[x.dtype], _FP4_FORMAT[fmt], 1 if act is not None else 0, 1 if gate_first else 0, _p(ws), n)
    return q, s


def unpack_fp4(q: torch.Tensor):
    """Packed codes uint8 [.., K/2] -> their values as e4m3 [.., K] (every e2m1 value is one)."""
    if q.dtype != torch.uint8 or not q.is_cuda or not q.is_contiguous() or q.dim() == 0 or q.shape[-1] % 8:
        raise ValueError("q must be a contiguous uint8 CUDA tensor whose last dimension is a multiple of 8")
    out = q.new_empty((*q.shape[:-1], 2 * q.shape[-1]), dtype=torch.float8_e4m3fn)
    _launch(_lib.UNPACK_FP4, q.device, q.data_ptr(), out.data_ptr(), q.numel())
    return out
