"""ctypes binding of the C ABI in ``include/b200moe.h``.

There is no fallback: if the CUDA library has not been built the import of any operator fails
with an error that says how to build it.
"""
from __future__ import annotations

import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libb200moe.so")

_c = ctypes


class GGArgs(_c.Structure):
    """``moe_gg_args`` of include/b200moe.h."""
    _fields_ = [
        ("a", _c.c_void_p), ("b", _c.c_void_p), ("sfa", _c.c_void_p),
        ("sfa_stride_row", _c.c_int64), ("sfa_stride_kblk", _c.c_int64),
        ("sfb", _c.c_void_p), ("layout", _c.c_void_p), ("d", _c.c_void_p), ("ldd", _c.c_int64),
        ("G", _c.c_int32), ("M", _c.c_int32), ("N", _c.c_int32), ("K", _c.c_int32),
        ("d_dtype", _c.c_int32), ("rows_used", _c.c_void_p),
        ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
        ("scatter_meta", _c.c_void_p), ("scatter_base", _c.c_void_p * 8),
        ("sf_format", _c.c_int32), ("sfb_stride", _c.c_int64 * 3), ("lda", _c.c_int64),
        ("ldb", _c.c_int64), ("accumulate", _c.c_int32), ("scatter_meta_stride", _c.c_int64),
        ("mx_tile", _c.c_int32),
    ]


class LayerArgs(_c.Structure):
    """``moe_layer_args`` of include/b200moe.h."""
    _fields_ = [
        ("x_q", _c.c_void_p), ("x_scale", _c.c_void_p), ("xs_stride_row", _c.c_int64), ("xs_stride_blk", _c.c_int64),
        ("logits", _c.c_void_p), ("topk_ids", _c.c_void_p), ("topk_weights", _c.c_void_p),
        ("w13", _c.c_void_p), ("w13_scale", _c.c_void_p), ("w2", _c.c_void_p), ("w2_scale", _c.c_void_p),
        ("out", _c.c_void_p), ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
        ("T", _c.c_int32), ("H", _c.c_int32), ("I", _c.c_int32), ("E", _c.c_int32), ("E_global", _c.c_int32),
        ("e_lo", _c.c_int32), ("top_k", _c.c_int32), ("align", _c.c_int32), ("gate_first", _c.c_int32),
        ("fuse_act", _c.c_int32), ("routing_bias", _c.c_void_p), ("n_group", _c.c_int32), ("topk_group", _c.c_int32),
        ("routed_scaling_factor", _c.c_float),
    ]


class LayerView(_c.Structure):
    """``moe_layer_view`` of include/b200moe.h."""
    _fields_ = [(n, _c.c_void_p) for n in ("ids", "counts", "offsets", "pos", "src_pair", "grouped_layout",
                                           "weights", "s1", "s2", "a1", "g1", "a2", "y")] + [("cap_rows", _c.c_int64)]


class KgArgs(_c.Structure):
    """``moe_kg_args`` of include/b200moe.h."""
    _fields_ = [
        ("a", _c.c_void_p), ("b", _c.c_void_p), ("sfa", _c.c_void_p), ("sfb", _c.c_void_p), ("d", _c.c_void_p),
        ("ks", _c.POINTER(_c.c_int32)), ("G", _c.c_int32), ("M", _c.c_int32), ("N", _c.c_int32), ("K_total", _c.c_int64),
        ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
    ]


class AlphaArgs(_c.Structure):
    """``moe_alpha_args`` of include/b200moe.h."""
    _fields_ = [
        ("hidden", _c.c_void_p), ("topk_ids", _c.c_void_p), ("topk_weights", _c.c_void_p),
        ("w13", _c.c_void_p), ("w13_scale", _c.c_void_p), ("w2", _c.c_void_p), ("w2_scale", _c.c_void_p),
        ("out", _c.c_void_p),
        ("M", _c.c_int32), ("H", _c.c_int32), ("I", _c.c_int32), ("E", _c.c_int32), ("top_k", _c.c_int32),
        ("routed_scaling_factor", _c.c_float), ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
    ]


class AlphaView(_c.Structure):
    """``moe_alpha_view`` of include/b200moe.h."""
    _fields_ = [(n, _c.c_void_p) for n in ("counts", "rowpos", "s1", "s2", "g1", "d2", "a1", "a2")] + [("max_m", _c.c_int64)]


class NormArgs(_c.Structure):
    """``moe_norm_args`` of include/b200moe.h."""
    _fields_ = [
        ("x", _c.c_void_p), ("x_stride", _c.c_int64), ("residual", _c.c_void_p), ("residual_stride", _c.c_int64),
        ("weight", _c.c_void_p), ("q", _c.c_void_p), ("scales", _c.c_void_p), ("ss_row", _c.c_int64), ("ss_blk", _c.c_int64),
        ("h", _c.c_void_p), ("y", _c.c_void_p), ("rstd", _c.c_void_p),
        ("T", _c.c_int32), ("H", _c.c_int32), ("dtype", _c.c_int32), ("w_dtype", _c.c_int32), ("pow2", _c.c_int32),
        ("eps", _c.c_float),
    ]


class NormGradArgs(_c.Structure):
    """``moe_norm_grad_args`` of include/b200moe.h."""
    _fields_ = [
        ("dy", _c.c_void_p), ("dy_stride", _c.c_int64), ("h", _c.c_void_p), ("h_stride", _c.c_int64),
        ("weight", _c.c_void_p), ("rstd", _c.c_void_p), ("dh", _c.c_void_p), ("dh_stride", _c.c_int64),
        ("dx", _c.c_void_p), ("dw", _c.c_void_p),
        ("T", _c.c_int32), ("H", _c.c_int32), ("dtype", _c.c_int32), ("w_dtype", _c.c_int32),
        ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
    ]


class RouteArgs(_c.Structure):
    """``moe_route_args`` of include/b200moe.h."""
    _fields_ = [
        ("logits", _c.c_void_p), ("stride", _c.c_int64), ("bias", _c.c_void_p), ("ids", _c.c_void_p), ("weights", _c.c_void_p),
        ("T", _c.c_int32), ("E", _c.c_int32), ("top_k", _c.c_int32), ("n_group", _c.c_int32), ("topk_group", _c.c_int32),
        ("dtype", _c.c_int32), ("bias_dtype", _c.c_int32), ("score", _c.c_int32), ("group_score", _c.c_int32),
        ("renormalize", _c.c_int32), ("scale", _c.c_float),
    ]


class RouteGradArgs(_c.Structure):
    """``moe_route_grad_args`` of include/b200moe.h."""
    _fields_ = [
        ("grad_weights", _c.c_void_p), ("logits", _c.c_void_p), ("stride", _c.c_int64), ("ids", _c.c_void_p),
        ("dlogits", _c.c_void_p), ("T", _c.c_int32), ("E", _c.c_int32), ("top_k", _c.c_int32), ("dtype", _c.c_int32),
        ("score", _c.c_int32), ("renormalize", _c.c_int32), ("scale", _c.c_float),
    ]


class Fp4QuantArgs(_c.Structure):
    """``moe_fp4_quant_args`` of include/b200moe.h."""
    _fields_ = [
        ("x", _c.c_void_p), ("x_stride", _c.c_int64), ("factor", _c.c_void_p), ("factor_stride", _c.c_int32),
        ("src_pair", _c.c_void_p), ("q", _c.c_void_p), ("scales", _c.c_void_p),
        ("groups", _c.c_int32), ("rows", _c.c_int32), ("src_rows", _c.c_int32), ("K", _c.c_int32), ("top_k", _c.c_int32),
        ("dtype", _c.c_int32), ("format", _c.c_int32), ("silu_mul", _c.c_int32), ("gate_first", _c.c_int32),
        ("workspace", _c.c_void_p), ("workspace_bytes", _c.c_uint64),
    ]


class GGFp4Args(_c.Structure):
    """``moe_gg_fp4_args`` of include/b200moe.h."""
    _fields_ = [
        ("a", _c.c_void_p), ("sfa", _c.c_void_p), ("b", _c.c_void_p), ("sfb", _c.c_void_p), ("alpha", _c.c_void_p),
        ("alpha_stride", _c.c_int32), ("layout", _c.c_void_p), ("rows_used", _c.c_void_p), ("d", _c.c_void_p),
        ("ldd", _c.c_int64), ("G", _c.c_int32), ("M", _c.c_int32), ("N", _c.c_int32), ("K", _c.c_int32),
        ("format", _c.c_int32), ("d_dtype", _c.c_int32),
    ]


class EpPeers(_c.Structure):
    """``moe_ep_peers`` of include/b200moe.h."""
    _fields_ = [("a", _c.c_void_p * 8), ("sa", _c.c_void_p * 8), ("y", _c.c_void_p * 8),
                ("counts", _c.c_void_p * 8), ("flags", _c.c_void_p * 8), ("meta", _c.c_void_p * 8)]


class EpSendArgs(_c.Structure):
    """``moe_ep_send_args`` of include/b200moe.h."""
    _fields_ = [("peers", _c.POINTER(EpPeers)), ("x_q", _c.c_void_p), ("x_scale", _c.c_void_p),
                ("xs_row", _c.c_int64), ("xs_blk", _c.c_int64), ("ids", _c.c_void_p), ("pos", _c.c_void_p),
                ("send_order", _c.c_void_p), ("counts_local", _c.c_void_p), ("n_pairs", _c.c_int64), ("pitch", _c.c_int64),
                ("top_k", _c.c_int32), ("E_local", _c.c_int32), ("H", _c.c_int32), ("cap_rows", _c.c_int32),
                ("rank", _c.c_int32), ("world", _c.c_int32)]


class B200MoeError(RuntimeError):
    pass


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise B200MoeError(
                f"{LIB_PATH} is missing: build it with `python -m tirx_harness_b200.build` "
                "(there is no CPU or PyTorch fallback)")
        _lib = ctypes.CDLL(LIB_PATH)
        _lib.moe_last_error.restype = _c.c_char_p
        _lib.moe_version.restype = _c.c_char_p
        for name in EXPORTS:
            fn = getattr(_lib, name)      # raises AttributeError if the symbol is absent
            if name in _SIZE_T_RETURN:
                fn.restype = _c.c_size_t
            elif name not in ("moe_last_error", "moe_version"):
                fn.restype = _c.c_int
    return _lib


# every symbol include/b200moe.h declares
EXPORTS = (
    "moe_gg_fp8_contiguous", "moe_gg_fp8_masked", "moe_gg_fp8_gate_up_act", "moe_gg_workspace_bytes", "moe_quant_1x128", "moe_silu_mul_requant",
    "moe_route_topk", "moe_route_deepseek", "moe_permute_workspace_bytes", "moe_permute_plan", "moe_permute_plan_static", "moe_permute",
    "moe_combine",
    "moe_rms_norm_quant", "moe_rms_norm_backward_workspace_bytes", "moe_rms_norm_backward", "moe_route", "moe_route_backward",
    "moe_quant_fp4", "moe_quant_fp4_workspace_bytes", "moe_unpack_fp4", "moe_gg_fp4_contiguous", "moe_gg_fp4_masked",
    "moe_workspace_bytes", "moe_layer_forward", "moe_layer_workspace_view", "moe_device_status",
    "moe_alpha_workspace_bytes", "moe_alpha_forward", "moe_alpha_workspace_view",
    "moe_kg_workspace_bytes", "moe_kg_fp8_contiguous",
    "moe_ipc_alloc", "moe_ipc_free", "moe_ipc_get_handle", "moe_ipc_open", "moe_ipc_close",
    "moe_ep_barrier", "moe_ep_workspace_bytes", "moe_ep_count_publish", "moe_ep_plan", "moe_ep_dispatch",
    "moe_ep_combine", "moe_ep_gate_up_dispatch", "moe_set_option", "moe_get_option",
    "moe_last_error", "moe_version",
)
_SIZE_T_RETURN = ("moe_gg_workspace_bytes", "moe_permute_workspace_bytes", "moe_workspace_bytes", "moe_ep_workspace_bytes",
                  "moe_alpha_workspace_bytes", "moe_kg_workspace_bytes", "moe_rms_norm_backward_workspace_bytes",
                  "moe_quant_fp4_workspace_bytes")


# dtypes and modes of include/b200moe.h
DTYPE_BF16, DTYPE_F32, DTYPE_F16 = range(3)
FP4_NV, FP4_MX = range(2)


# moe_set_option keys and values (include/b200moe.h)
OPT_GG_BLOCK_SCALED, OPT_MX_TILE, OPT_ALPHA_PATH, OPT_ALPHA_GEMV_MAX_ROUTES, OPT_KG_MODE, OPT_EP_WAIT_LIMIT_MS = range(6)
MX_TILE_AUTO, MX_TILE_PAIR, MX_TILE_SINGLE, MX_TILE_PAIR_240, MX_TILE_PAIR_224 = range(5)
ALPHA_PATH_AUTO, ALPHA_PATH_SWAP, ALPHA_PATH_MASKED, ALPHA_PATH_MIXED = range(4)
KG_MODE_MN_MAJOR, KG_MODE_TRANSPOSE, KG_MODE_PER_GROUP = range(3)


def set_option(option: int, value: int) -> int:
    """Sets a process-wide mode and returns the previous value (so a caller can restore it)."""
    old = ctypes.c_int32(0)
    check(lib().moe_get_option(ctypes.c_int32(option), ctypes.byref(old)))
    check(lib().moe_set_option(ctypes.c_int32(option), ctypes.c_int32(value)))
    return old.value


class Entry:
    """An entry point that takes one argument block and a stream.  ``pack`` lays a block's values out as bytes in the order
    of the structure's fields (pointers as integers, 0 = NULL), several times faster than filling a ctypes structure: a
    call that launches one small kernel costs the host more than the GPU."""

    _CODES = {_c.c_void_p: "P", _c.c_int64: "q", _c.c_uint64: "Q", _c.c_int32: "i", _c.c_float: "f"}
    _ARGTYPES = (_c.c_char_p, _c.c_void_p)

    def __init__(self, name: str, args):
        layout = struct.Struct("@" + "".join(self._CODES[t] for _, t in args._fields_) + "0P")
        assert layout.size == _c.sizeof(args), name
        self.pack, self._name, self._fn, self._fields = layout.pack, name, None, args._fields_

    def misfit(self, values) -> Exception:
        """What is wrong with values that ``pack`` could not lay out."""
        for (field, kind), v in zip(self._fields, values):
            try:
                struct.pack("@" + self._CODES[kind], v)
            except OverflowError:
                return ValueError(f"{field}={v} does not fit its {_c.sizeof(kind) * 8} bits")
            except struct.error:
                if hasattr(v, "__index__"):
                    return ValueError(f"{field}={v} does not fit its {_c.sizeof(kind) * 8} bits")
                return TypeError(f"{field} must be {'a number' if kind is _c.c_float else 'an integer'}, got {v!r}")
        return TypeError(f"{self._name} takes {len(self._fields)} values, got {len(values)}")

    def _bind(self):
        self._fn = _c.CFUNCTYPE(_c.c_int, *self._ARGTYPES)((self._name, lib()))
        return self._fn

    def __call__(self, block: bytes, stream: int) -> None:
        rc = (self._fn or self._bind())(block, stream)
        if rc != 0:
            check(rc)


class UnpackEntry(Entry):
    """moe_unpack_fp4: pointers and a size instead of a block."""

    _ARGTYPES = (_c.c_void_p, _c.c_void_p, _c.c_int64, _c.c_void_p)

    def __init__(self, name: str):
        self.pack, self._name, self._fn = (lambda *values: values), name, None

    def __call__(self, values, stream: int) -> None:
        rc = (self._fn or self._bind())(*values, stream)
        if rc != 0:
            check(rc)


NORM = Entry("moe_rms_norm_quant", NormArgs)
NORM_GRAD = Entry("moe_rms_norm_backward", NormGradArgs)
ROUTE = Entry("moe_route", RouteArgs)
ROUTE_GRAD = Entry("moe_route_backward", RouteGradArgs)
UNPACK_FP4 = UnpackEntry("moe_unpack_fp4")
FP4_QUANT = Entry("moe_quant_fp4", Fp4QuantArgs)
GG_FP4_CONTIGUOUS = Entry("moe_gg_fp4_contiguous", GGFp4Args)
GG_FP4_MASKED = Entry("moe_gg_fp4_masked", GGFp4Args)


def check(rc: int) -> None:
    if rc != 0:
        raise B200MoeError(f"b200moe error {rc}: {lib().moe_last_error().decode()}")
