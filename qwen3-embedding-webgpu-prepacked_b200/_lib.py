"""ctypes binding of libqwa.so (the C ABI in include/qwa.h).

There is no fallback: if the library is missing or cannot be loaded, every
call raises. Build it with ``build.build()`` (or ``__graft_entry__.build()``).
"""
from __future__ import annotations

import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libqwa.so")

QWA_OK, QWA_ERR_INVALID_ARG, QWA_ERR_UNSUPPORTED, QWA_ERR_CUDA, QWA_ERR_TIMEOUT, \
    QWA_ERR_NO_DEVICE = range(6)
MODE_AUTO, MODE_FULL, MODE_SPARSE = 0, 1, 2

P = ctypes.c_void_p
I32, I64, F32 = ctypes.c_int, ctypes.c_int64, ctypes.c_float
I32P = ctypes.POINTER(ctypes.c_int32)
I64P = ctypes.POINTER(ctypes.c_int64)

F64 = ctypes.c_double

# qwa_dtype, qwa_kv_format, qwa_rope_layout, qwa_rope_scaling_kind
DTYPE_F16, DTYPE_BF16 = 0, 1
KV_PLAIN, KV_E4M3, KV_INT8 = 0, 1, 2
ROPE_HALF, ROPE_INTERLEAVED = 0, 1
ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}


class RopeScalingStruct(ctypes.Structure):
    """qwa_rope_scaling"""
    _fields_ = [("kind", I32), ("factor", F64), ("original_positions", F64), ("beta_fast", F64),
                ("beta_slow", F64), ("attention_factor", F64), ("low_freq_factor", F64),
                ("high_freq_factor", F64)]


# qwa_rope_tensor and qwa_kv_cache as bytes, in the order of their fields: a call takes
# them as a pointer, and they are made in a quarter of a ctypes structure's time
rope_tensor = struct.Struct("@PqqPqqi4x").pack
kv_cache = struct.Struct("@iiiiqPPPP").pack

# name -> (restype, argtypes); the exported surface of include/qwa.h
SIGNATURES = {
    "qwa_create": (I32, [I32, ctypes.POINTER(P)]),
    "qwa_destroy": (I32, [P]),
    "qwa_last_error": (ctypes.c_char_p, [P]),
    "qwa_status_string": (ctypes.c_char_p, [I32]),
    "qwa_version": (ctypes.c_char_p, []),
    "qwa_qk_norm_rope": (I32, [P, P, I64, P, P, P, P, I32P, I32, F32, F32, P, P]),
    "qwa_qk_norm_rope_padded": (I32, [P, P, I64, P, P, P, P, I32, I32, F32, F32, P, P]),
    "qwa_attention": (I32, [P, P, P, P, I64, I64, P, I32P, I32, I32, I32, I32, P]),
    "qwa_attention_padded": (I32, [P, P, P, P, P, I32, I32, I32, I32, I64, I64, P]),
    "qwa_prefill_attention_layer": (I32, [P, P, I64, P, P, P, P, P, I32P, I32, I32, I32, I32, F32,
                                          F32, P]),
    "qwa_check": (I32, [P, P]),
    "qwa_set_debug": (I32, [P, I64, I32]),
    "qwa_attention_work": (I32, [I32P, I32, I32, I32, I32, I64P, I64P]),
    "qwa_selftest_tile": (I32, [P, P, P, P, P, P, P]),
    "qwa_attention_noalloc": (I32, [P, P, P, I64, I64, P, I32P, I32, I32, I32, I32, P]),
    "qwa_matmul": (I32, [P, P, P, P, I32, I32, I32, P]),
    "qwa_matmul_swiglu": (I32, [P, P, P, P, I32, I32, I32, P]),
    "qwa_q40_dequantize": (I32, [P, P, I32, I32, P, P]),
    "qwa_q40_matmul": (I32, [P, P, P, P, I32, I32, I32, P]),
    "qwa_q40_forget": (I32, [P, P]),
    "qwa_qkv_projection": (I32, [P, P, P, I32, P, P, P, P, P, I32P, I32, F32, F32, P, P]),
    "qwa_q40_qkv_projection": (I32, [P, P, P, I32, P, P, P, P, P, I32P, I32, F32, F32, P, P]),
    "qwa_rms_norm": (I32, [P, P, P, P, P, I32, I32, F32, I32, P]),
    "qwa_swiglu": (I32, [P, P, P, I32, I32, P]),
    "qwa_embedding_lookup_q6k": (I32, [P, P, P, I32, P, I32, I32, P]),
    "qwa_last_token_pool": (I32, [P, P, I32, P, I32P, I32, P]),
    "qwa_last_token_pool_padded": (I32, [P, P, P, P, I32, I32, I32, P]),
    "qwa_rope_table": (I32, [P, P, I64, I32, I32, F64, ctypes.POINTER(RopeScalingStruct), P]),
    "qwa_rope": (I32, [P, I32, P, P, I32, I32, I32, I32, I32, P, P, I32, P]),
    "qwa_kv_cache_write": (I32, [P, P, P, I64, P, I64, P, I32, P]),
    "qwa_kv_cache_read": (I32, [P, P, P, I32, P, P, P]),
    "qwa_prefix_plan_create": (I32, [P, I32P, I32P, I32, I32, I32, I32, I32, I32, I32,
                                     ctypes.POINTER(P)]),
    "qwa_prefix_plan_destroy": (I32, [P]),
    "qwa_prefix_plan_deal": (I32, [P, ctypes.POINTER(I32), ctypes.POINTER(I32)]),
    "qwa_prefix_attention_workspace": (ctypes.c_size_t, [P, I32]),
    "qwa_prefix_attention": (I32, [P, P, I32, P, I64, P, I64, P, I64, P, P, I64, P,
                                   ctypes.c_size_t, P]),
    "qwa_prefix_attention_work": (I32, [I32P, I32P, I32, I32, I32, I32, I32, I32, I32, I64P,
                                        I64P]),
}

_lib = None


class QwaError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"qwa status {status}: {message}")
        self.status = status


def load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built; run the package's build.build() first")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def status_string(status: int) -> str:
    return load().qwa_status_string(status).decode()


def check(status: int, ctx=None) -> None:
    if status != QWA_OK:
        msg = load().qwa_last_error(ctx).decode() if ctx else ""
        raise QwaError(status, msg or status_string(status))


def cu_array(cu_seqlens) -> ctypes.Array:
    vals = [int(x) for x in cu_seqlens]
    return (ctypes.c_int32 * len(vals))(*vals)
