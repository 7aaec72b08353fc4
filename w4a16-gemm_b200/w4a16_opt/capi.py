"""ctypes binding of the C ABI (include/w4a16.h) -- the binding a non-torch host adds.

    lib = load()                         # libw4a16.so next to this file
    st = lib.w4a16_gemm(Wp_ptr, x_ptr, s_ptr, y_ptr, M, N, K, groups, wp_words,
                        variant, W4A16_OUT_F16, ws_ptr, ws_bytes, stream_ptr)

Every exported function and its argument types are declared here; the
``EXPORTS`` table is the list include/w4a16.h declares.
"""
from __future__ import annotations

import ctypes
import os

W4A16_OK = 0
W4A16_OUT_F16 = 0
W4A16_OUT_F32 = 1
W4A16_FLAG_WEIGHTS_RESIDENT = 1
W4A16_FLAG_FP32_SCALE = 2

STATUS_NAMES = {
    0: "W4A16_OK", 1: "W4A16_ERR_NULL_POINTER", 2: "W4A16_ERR_VARIANT", 3: "W4A16_ERR_M",
    4: "W4A16_ERR_DIM_RANGE", 5: "W4A16_ERR_K_MULTIPLE", 6: "W4A16_ERR_N_MULTIPLE", 7: "W4A16_ERR_GROUPS",
    8: "W4A16_ERR_WP_SIZE", 9: "W4A16_ERR_ALIGNMENT", 10: "W4A16_ERR_GROUP_SIZE",
    11: "W4A16_ERR_DECODE_SHAPE", 12: "W4A16_ERR_OUT_DTYPE", 13: "W4A16_ERR_DEVICE", 14: "W4A16_ERR_CUDA",
    15: "W4A16_ERR_DEVICE_TIMEOUT", 16: "W4A16_ERR_WORKSPACE", 17: "W4A16_ERR_FLAGS", 18: "W4A16_ERR_TP_GROUP",
    19: "W4A16_ERR_CACHE", 20: "W4A16_ERR_ACT_DTYPE",
    21: "W4A16_ERR_ACTIVATION", 22: "W4A16_ERR_OVERLAP", 23: "W4A16_ERR_NORM", 24: "W4A16_ERR_MOE",
}
TP_MAX_RANKS = 8
TP_CTRL_BYTES = 8192
TP_PUSH_MAX_BYTES = 1 << 20


class Route(ctypes.Structure):
    _fields_ = [(name, ctypes.c_int32) for name in
                ("kernel", "config", "tile_m", "tile_n", "split_k", "grid", "stages", "smem_bytes")] + \
               [("workspace_bytes", ctypes.c_uint64), ("launches", ctypes.c_int32), ("reserved", ctypes.c_int32)]


_i64, _i32, _u64, _vp = ctypes.c_int64, ctypes.c_int32, ctypes.c_uint64, ctypes.c_void_p


class IpcHandle(ctypes.Structure):
    _fields_ = [("bytes", ctypes.c_ubyte * 64)]


class TpGroup(ctypes.Structure):
    _fields_ = [("rank", ctypes.c_int32), ("world", ctypes.c_int32), ("buf", ctypes.c_void_p * TP_MAX_RANKS),
                ("buf_bytes", ctypes.c_uint64), ("recv_off", ctypes.c_uint64), ("recv_bytes", ctypes.c_uint64)]


class Cache(ctypes.Structure):
    """w4a16_cache: a paged 4-bit key/value cache."""
    _fields_ = [("data", _vp), ("num_pages", _i64), ("page_size", _i32), ("kv_heads", _i32), ("head_dim", _i32),
                ("group_size", _i32)]


class Rotary(ctypes.Structure):
    """w4a16_rotary: positions and tables of an append's rotary embedding."""
    _fields_ = [("q", _vp), ("q_out", _vp), ("q_token_stride", _i64), ("q_head_stride", _i64), ("positions", _vp),
                ("positions_axis_stride", _i64), ("cos_sin", _vp), ("max_pos", _i64), ("q_heads", _i32),
                ("axes", _i32), ("sections", _i32 * 3), ("rotary_dim", _i32), ("interleaved", _i32)]


class CacheAttentionArgs(ctypes.Structure):
    """w4a16_cache_attention_args: one attention call over a cache."""
    _fields_ = [("q", _vp), ("out", _vp), ("lse", _vp), ("q_token_stride", _i64), ("q_head_stride", _i64),
                ("q_tokens", _i64), ("page_table", _vp), ("page_table_stride", _i64), ("seq_lens", _vp), ("cu_q", _vp),
                ("scale", ctypes.c_float), ("dtype", _i32), ("q_heads", _i32), ("batch", _i32), ("table_pages", _i32),
                ("max_q", _i32), ("causal", _i32), ("window", _i32)]


class Epilogue(ctypes.Structure):
    """w4a16_epilogue: what w4a16_linear does with a product's sums."""
    _fields_ = [("bias", _vp), ("residual", _vp), ("activation", _i32), ("gated", _i32)]


class NormArgs(ctypes.Structure):
    """w4a16_norm_args: one w4a16_rms_norm call."""
    _fields_ = [("x", _vp), ("weight", _vp), ("residual", _vp), ("y", _vp), ("residual_out", _vp)] + \
               [(f"{name}_{axis}_stride", _i64) for name in ("x", "residual", "y", "residual_out") for axis in ("token", "head")] + \
               [("tokens", _i64), ("heads", _i32), ("dim", _i32), ("dtype", _i32), ("residual_f32", _i32),
                ("eps", ctypes.c_float)]


class MoeArgs(ctypes.Structure):
    """w4a16_moe_args: one w4a16_moe_experts call."""
    _fields_ = [(name, _vp) for name in ("x", "gate_up_wp", "gate_up_scales", "down_wp", "down_scales", "experts", "weights",
                                         "residual", "y")] + [("tokens", _i64)] + \
               [(name, _i32) for name in ("num_experts", "k", "hidden", "inner", "gate_up_group", "down_group", "activation")]


# name -> (restype, argtypes), one entry per declaration in include/w4a16.h
EXPORTS = {
    "w4a16_abi_version": (_i32, []),
    "w4a16_validate": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32]),
    "w4a16_workspace_bytes": (_i32, [_i64, _i64, _i64, _i64, _i32, ctypes.POINTER(_u64)]),
    "w4a16_gemm": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _vp, _u64, _vp]),
    "w4a16_gemm_ex": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _i32, ctypes.c_uint32, _vp,
                             _u64, _vp]),
    "w4a16_gemm_noalloc": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _vp]),
    "w4a16_query_route": (_i32, [_i64, _i64, _i64, _i64, _i32, ctypes.POINTER(Route)]),
    "w4a16_dequant": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _vp]),
    "w4a16_pack": (_i32, [_vp, _vp, _i64, _i64, _vp]),
    "w4a16_quantize": (_i32, [_vp, _i32, _vp, _vp, _i64, _i64, _i64, _vp]),
    "w4a16_quantize_pack": (_i32, [_vp, _i32, _vp, _vp, _i64, _i64, _i64, _vp]),
    "w4a16_peer_alloc": (_i32, [_u64, ctypes.POINTER(_vp), ctypes.POINTER(IpcHandle)]),
    "w4a16_peer_open": (_i32, [ctypes.POINTER(IpcHandle), ctypes.POINTER(_vp)]),
    "w4a16_peer_close": (_i32, [_vp]),
    "w4a16_peer_free": (_i32, [_vp]),
    "w4a16_tp_allreduce": (_i32, [ctypes.POINTER(TpGroup), _u64, _u64, _i64, _i64, _vp]),
    "w4a16_tp_allgather": (_i32, [ctypes.POINTER(TpGroup), _u64, _u64, _i64, _i64, _vp]),
    "w4a16_cache_page_bytes": (_i32, [_i32, _i32, _i32, ctypes.POINTER(_u64)]),
    "w4a16_cache_append": (_i32, [ctypes.POINTER(Cache), _vp, _vp, _i64, _i64, _i64, _i64, _i32, _vp, _i64,
                                  ctypes.POINTER(Rotary), _vp]),
    "w4a16_cache_read": (_i32, [ctypes.POINTER(Cache), _vp, _i64, _vp, _vp, _i32, _vp]),
    "w4a16_cache_attention": (_i32, [ctypes.POINTER(Cache), ctypes.POINTER(CacheAttentionArgs), _vp, _u64, _vp]),
    "w4a16_cache_attention_workspace": (_i32, [ctypes.POINTER(Cache), ctypes.POINTER(CacheAttentionArgs),
                                               ctypes.POINTER(_u64)]),
    "w4a16_linear": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, ctypes.POINTER(Epilogue), _i32,
                            ctypes.c_uint32, _vp, _u64, _vp]),
    "w4a16_rms_norm": (_i32, [ctypes.POINTER(NormArgs), _vp]),
    "w4a16_moe_route": (_i32, [_vp, _i32, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp]),
    "w4a16_moe_experts": (_i32, [ctypes.POINTER(MoeArgs), _vp, _u64, _vp]),
    "w4a16_moe_workspace": (_i32, [ctypes.POINTER(MoeArgs), ctypes.POINTER(_u64)]),
    "w4a16_device_status": (_i32, [ctypes.POINTER(_i32), _i32]),
    "w4a16_check_wait_limits": (_i32, [ctypes.POINTER(_i32)]),
    "w4a16_status_string": (ctypes.c_char_p, [_i32]),
    "w4a16_last_error": (ctypes.c_char_p, []),
}

_LIB = None


def library_path() -> str:
    return os.path.join(os.path.dirname(os.path.abspath(__file__)), "libw4a16.so")


def load(path: str | None = None) -> ctypes.CDLL:
    """Load libw4a16.so and declare every exported signature."""
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    lib = ctypes.CDLL(path or library_path())
    for name, (res, args) in EXPORTS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if path is None:
        _LIB = lib
    return lib


def last_error(lib: ctypes.CDLL | None = None) -> str:
    lib = lib or load()
    return lib.w4a16_last_error().decode()


class W4A16Error(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"{STATUS_NAMES.get(status, status)}: {message}")
        self.status = status


def check(status: int, lib: ctypes.CDLL | None = None) -> None:
    if status != W4A16_OK:
        raise W4A16Error(status, last_error(lib))
