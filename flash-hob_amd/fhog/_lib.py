"""ctypes binding of ``libfhog_hip.so`` (C ABI in ``include/fhog_hip.h``).

The library is loaded from this directory.  It is never built implicitly at import time
on a machine with a GPU and there is no other implementation to fall back to: if the
shared object is missing, :func:`lib` raises.
"""
from __future__ import annotations

import ctypes
from ctypes import POINTER, Structure, c_char_p, c_double, c_float, c_int, c_int32, c_int64, c_size_t, c_void_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libfhog_hip.so"

DTYPE_BF16, DTYPE_FP32, DTYPE_FP16 = 0, 1, 2
POSITIONS_INT32, POSITIONS_INT64, POSITIONS_FP32 = 0, 1, 2
ROTARY_MAX_D, ROTARY_MAX_AXES = 256, 4
IMPL_AUTO, IMPL_FP32, IMPL_BF16 = 0, 1, 2
MASK_NONE, MASK_TOP_LEFT, MASK_BOTTOM_RIGHT = 0, 1, 2
PASS_D, PASS_DD, PASS_B, PASS_DQ_DDO, PASS_DK_DV, PASS_DD_B, PASS_B_DDO, PASS_DQ, PASS_DD_B_DDO, PASS_STAGE1 = range(10)
SCHEDULE_FOUR_PASS, SCHEDULE_FUSED_STATS, SCHEDULE_DDO_EARLY, SCHEDULE_THREE_SWEEP = range(4)
ABI_VERSION = 5
STATIC_WS_BYTES = 16 << 20   # of a default build; `lib().fhog_static_ws_bytes()` tells what the loaded library holds

ERROR_NAMES = {
    -1: "FHOG_E_NULL", -2: "FHOG_E_SHAPE", -3: "FHOG_E_DTYPE", -4: "FHOG_E_STRIDE", -5: "FHOG_E_ALIGN",
    -6: "FHOG_E_CAUSAL", -7: "FHOG_E_PASS", -8: "FHOG_E_LAUNCH", -9: "FHOG_E_SCALE", -10: "FHOG_E_IMPL",
    -11: "FHOG_E_SCHEDULE", -12: "FHOG_E_ROTARY", -13: "FHOG_E_PAGED",
}


class BwdBwdArgs(Structure):
    """Mirror of ``fhog_bwdbwd_args``."""
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("o", c_void_p), ("dO", c_void_p),
        ("ddq", c_void_p), ("ddk", c_void_p), ("ddv", c_void_p), ("lse", c_void_p),
        ("dq2", c_void_p), ("dk2", c_void_p), ("dv2", c_void_p), ("ddo", c_void_p), ("ws", c_void_p),
        ("batch", c_int64), ("n_q", c_int64), ("n_k", c_int64), ("d", c_int64),
        ("stride_qb", c_int64), ("stride_qn", c_int64), ("stride_kb", c_int64), ("stride_kn", c_int64),
        ("scale", c_float), ("dtype", c_int32), ("causal", c_int32), ("impl", c_int32), ("schedule", c_int32),
        ("window", c_int64), ("ws_bytes", c_int64),
    ]


class AttnArgs(Structure):
    """Mirror of ``fhog_attn_args``."""
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("o", c_void_p), ("lse", c_void_p),
        ("dO", c_void_p), ("dq", c_void_p), ("dk", c_void_p), ("dv", c_void_p), ("ws", c_void_p),
        ("batch", c_int64), ("n_q", c_int64), ("n_k", c_int64), ("d", c_int64),
        ("stride_qb", c_int64), ("stride_qn", c_int64), ("stride_kb", c_int64), ("stride_kn", c_int64),
        ("scale", c_float), ("dtype", c_int32), ("causal", c_int32), ("window", c_int32),
    ]


class RotaryArgs(Structure):
    """Mirror of ``fhog_rotary_args``."""
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("q_out", c_void_p), ("k_out", c_void_p), ("positions", c_void_p),
        ("batch", c_int64), ("heads_q", c_int64), ("heads_k", c_int64), ("n", c_int64), ("d", c_int64), ("rotary_dim", c_int64),
        ("stride_qb", c_int64), ("stride_qh", c_int64), ("stride_qn", c_int64), ("stride_kb", c_int64), ("stride_kh", c_int64), ("stride_kn", c_int64),
        ("stride_qob", c_int64), ("stride_qoh", c_int64), ("stride_qon", c_int64), ("stride_kob", c_int64), ("stride_koh", c_int64),
        ("stride_kon", c_int64), ("stride_pa", c_int64), ("stride_pb", c_int64), ("stride_pn", c_int64),
        ("theta", c_double), ("sections", c_int32 * 4), ("axes", c_int32), ("dtype", c_int32), ("position_type", c_int32), ("interleaved", c_int32),
        ("inverse", c_int32),
    ]


class PagedCacheArgs(Structure):
    """Mirror of ``fhog_paged_cache``."""
    _fields_ = [
        ("keys", c_void_p), ("values", c_void_p), ("table", c_void_p), ("lengths", c_void_p),
        ("batch", c_int64), ("heads_k", c_int64), ("d", c_int64), ("pages", c_int64), ("page", c_int64), ("table_width", c_int64),
        ("stride_p", c_int64), ("stride_h", c_int64), ("stride_n", c_int64), ("stride_tb", c_int64), ("dtype", c_int32),
    ]


class PagedAppendArgs(Structure):
    """Mirror of ``fhog_paged_append_args``."""
    _fields_ = [
        ("cache", PagedCacheArgs), ("k", c_void_p), ("v", c_void_p), ("counts", c_void_p), ("n", c_int64),
        ("stride_kb", c_int64), ("stride_kh", c_int64), ("stride_kn", c_int64), ("stride_vb", c_int64), ("stride_vh", c_int64), ("stride_vn", c_int64),
    ]


class PagedAttnArgs(Structure):
    """Mirror of ``fhog_paged_attn_args``."""
    _fields_ = [
        ("cache", PagedCacheArgs), ("q", c_void_p), ("o", c_void_p), ("lse", c_void_p), ("weights_in", c_void_p), ("weights_out", c_void_p), ("ws", c_void_p),
        ("heads_q", c_int64), ("stride_qb", c_int64), ("stride_qh", c_int64), ("stride_ob", c_int64), ("stride_oh", c_int64),
        ("stride_wib", c_int64), ("stride_wih", c_int64), ("stride_wob", c_int64), ("stride_woh", c_int64), ("window", c_int64), ("sinks", c_int64),
        ("ws_bytes", c_int64), ("scale", c_float),
    ]


class KeyWeightsArgs(Structure):
    """Mirror of ``fhog_key_weights_args``."""
    _fields_ = [
        ("q", c_void_p), ("k", c_void_p), ("lse", c_void_p), ("lengths", c_void_p), ("out", c_void_p), ("ws", c_void_p),
        ("batch", c_int64), ("heads_q", c_int64), ("heads_k", c_int64), ("n_q", c_int64), ("n_k", c_int64), ("d", c_int64),
        ("stride_qb", c_int64), ("stride_qh", c_int64), ("stride_qn", c_int64), ("stride_kb", c_int64), ("stride_kh", c_int64), ("stride_kn", c_int64),
        ("stride_ob", c_int64), ("stride_oh", c_int64), ("window", c_int64), ("sinks", c_int64), ("ws_bytes", c_int64),
        ("scale", c_float), ("dtype", c_int32), ("causal", c_int32),
    ]


class PagedEvictArgs(Structure):
    """Mirror of ``fhog_paged_evict_args``."""
    _fields_ = [
        ("cache", PagedCacheArgs), ("weights", c_void_p), ("into", c_void_p), ("lengths_out", c_void_p), ("kept", c_void_p), ("weights_out", c_void_p),
        ("stride_wb", c_int64), ("stride_wh", c_int64), ("stride_ib", c_int64), ("into_width", c_int64), ("budget", c_int64), ("sinks", c_int64), ("recent", c_int64),
    ]


class FhogError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{ERROR_NAMES.get(code, code)}: {message}")
        self.code = code


_LIB = None


def lib() -> ctypes.CDLL:
    """Load (once) and return the shared library; raise if it is not there."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python flash-hob_amd/fhog/build.py` "
            "(hipcc, gfx950). There is no fallback implementation.")
    L = ctypes.CDLL(str(LIB_PATH))
    L.fhog_abi_version.restype = c_int
    L.fhog_abi_version.argtypes = []
    L.fhog_bwdbwd_workspace_bytes.restype = c_size_t
    L.fhog_bwdbwd_workspace_bytes.argtypes = [c_int64, c_int64]
    L.fhog_bwdbwd_workspace_hint.restype = c_size_t
    L.fhog_bwdbwd_workspace_hint.argtypes = [POINTER(BwdBwdArgs)]
    L.fhog_validate.restype = c_int
    L.fhog_validate.argtypes = [POINTER(BwdBwdArgs)]
    L.fhog_select_impl.restype = c_int
    L.fhog_select_impl.argtypes = [POINTER(BwdBwdArgs)]
    L.fhog_bwdbwd.restype = c_int
    L.fhog_bwdbwd.argtypes = [POINTER(BwdBwdArgs), c_void_p]
    L.fhog_bwdbwd_static_ws.restype = c_int
    L.fhog_bwdbwd_static_ws.argtypes = [POINTER(BwdBwdArgs), c_void_p]
    L.fhog_static_ws_bytes.restype = c_size_t
    L.fhog_static_ws_bytes.argtypes = []
    L.fhog_bwdbwd_pass.restype = c_int
    L.fhog_bwdbwd_pass.argtypes = [POINTER(BwdBwdArgs), c_int, c_void_p]
    L.fhog_last_error.restype = c_char_p
    L.fhog_last_error.argtypes = []
    L.fhog_bwdbwd_args_size.restype = c_size_t
    L.fhog_bwdbwd_args_size.argtypes = []
    L.fhog_attn_args_size.restype = c_size_t
    L.fhog_attn_args_size.argtypes = []
    L.fhog_attn_validate.restype = c_int
    L.fhog_attn_validate.argtypes = [POINTER(AttnArgs), c_int]
    L.fhog_attn_fwd.restype = c_int
    L.fhog_attn_fwd.argtypes = [POINTER(AttnArgs), c_void_p]
    L.fhog_attn_bwd.restype = c_int
    L.fhog_attn_bwd.argtypes = [POINTER(AttnArgs), c_void_p]
    L.fhog_attn_sinks_workspace_bytes.restype = c_size_t
    L.fhog_attn_sinks_workspace_bytes.argtypes = [POINTER(AttnArgs), c_int64, c_int]
    L.fhog_attn_fwd_sinks.restype = c_int
    L.fhog_attn_fwd_sinks.argtypes = [POINTER(AttnArgs), c_int64, c_void_p, c_int64, c_void_p]
    L.fhog_attn_bwd_sinks.restype = c_int
    L.fhog_attn_bwd_sinks.argtypes = [POINTER(AttnArgs), c_int64, c_int64, c_void_p]
    L.fhog_bwdbwd_sinks_workspace_bytes.restype = c_size_t
    L.fhog_bwdbwd_sinks_workspace_bytes.argtypes = [POINTER(BwdBwdArgs), c_int64]
    L.fhog_bwdbwd_sinks.restype = c_int
    L.fhog_bwdbwd_sinks.argtypes = [POINTER(BwdBwdArgs), c_int64, c_void_p]
    L.fhog_rotary_args_size.restype = c_size_t
    L.fhog_rotary_args_size.argtypes = []
    L.fhog_rotary_validate.restype = c_int
    L.fhog_rotary_validate.argtypes = [POINTER(RotaryArgs)]
    L.fhog_rotary.restype = c_int
    L.fhog_rotary.argtypes = [POINTER(RotaryArgs), c_void_p]
    for call, args in (("paged_append", PagedAppendArgs), ("paged_attn", PagedAttnArgs), ("key_weights", KeyWeightsArgs), ("paged_evict", PagedEvictArgs)):
        size, validate, run = (getattr(L, f"fhog_{call}{x}") for x in ("_args_size", "_validate", ""))
        size.restype, size.argtypes = c_size_t, []
        validate.restype, validate.argtypes = c_int, [POINTER(args)]
        run.restype, run.argtypes = c_int, [POINTER(args), c_void_p]
        if size() != ctypes.sizeof(args):
            raise RuntimeError(f"fhog_{call}_args layout differs between libfhog_hip.so and the ctypes mirror")
    L.fhog_paged_attn_workspace_bytes.restype = L.fhog_key_weights_workspace_bytes.restype = c_size_t
    L.fhog_paged_attn_workspace_bytes.argtypes = [POINTER(PagedAttnArgs)]
    L.fhog_key_weights_workspace_bytes.argtypes = [POINTER(KeyWeightsArgs)]
    L.fhog_probe_mfma_rate.restype = c_int
    L.fhog_probe_mfma_rate.argtypes = [c_void_p, c_int, c_int, c_int, POINTER(ctypes.c_double), c_void_p]
    if L.fhog_attn_args_size() != ctypes.sizeof(AttnArgs):
        raise RuntimeError("fhog_attn_args layout differs between libfhog_hip.so and the ctypes mirror")
    if L.fhog_rotary_args_size() != ctypes.sizeof(RotaryArgs):
        raise RuntimeError("fhog_rotary_args layout differs between libfhog_hip.so and the ctypes mirror")
    if L.fhog_bwdbwd_args_size() != ctypes.sizeof(BwdBwdArgs):
        raise RuntimeError("fhog_bwdbwd_args layout differs between libfhog_hip.so and the ctypes mirror")
    if L.fhog_abi_version() != ABI_VERSION:
        raise RuntimeError(f"libfhog_hip.so ABI {L.fhog_abi_version()} != binding {ABI_VERSION}")
    _LIB = L
    return L


_TORCH_EXT = None


def torch_ext():
    """Load (once) and return the native host side of the PyTorch entry points; raise if it is not there."""
    global _TORCH_EXT
    if _TORCH_EXT is None:
        lib()
        try:
            from . import _fhog_torch
        except ImportError as why:
            raise RuntimeError("_fhog_torch.so is missing or does not load: build it with `python flash-hob_amd/fhog/build.py`") from why
        _TORCH_EXT = _fhog_torch
    return _TORCH_EXT


def check_memory(**tensors) -> None:
    """Raise on a tensor on a GPU whose storage holds no memory. A view of one that starts behind its first element has an address all the same."""
    for name, t in tensors.items():
        if t is not None and t.is_cuda and not torch_ext().in_memory(t):
            raise ValueError(f"{name} holds no memory (a fake tensor, or a storage that was resized to nothing)")


def check(rc: int) -> None:
    if rc != 0:
        raise FhogError(rc, lib().fhog_last_error().decode())
