"""ctypes binding of the C ABI in include/consumer_int8_amd.h, include/consumer_int8_attention.h
and include/consumer_int8_drafts.h (libci8_amd.so).

This is the binding an FFI caller would write; the torch ops do not use it (they call
the same entry points from C++). Tests use it to reach the C ABI directly.
"""

from __future__ import annotations

import ctypes
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libci8_amd.so"

CI8_OK = 0
CI8_ERR_GEOMETRY = 1
CI8_ERR_ALIGNMENT = 2
CI8_ERR_OVERLAP = 3
CI8_ERR_SCHEDULE = 4
CI8_ERR_TOO_LARGE = 5
CI8_ERR_LAUNCH = 6

_p = ctypes.c_void_p
_i64 = ctypes.c_int64

SIGNATURES = {
    "ci8_last_error": ([], ctypes.c_char_p),
    "ci8_version": ([], ctypes.c_char_p),
    "ci8_quantize_rows": ([_p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_quantize_grouped4096": ([_p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_fused_channel_mm": ([_p, _p, _p, _p, _p, _i64, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_cutlass_channel_mm": ([_p, _p, _p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_cutlass_channel_mm_noalloc": ([_p, _p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_channel_mm": ([_p, _p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_channel_gemv": ([_p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_grouped_summed_mm": ([_p, _p, _p, _p, _p, _i64, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_silu_mul": ([_p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_silu_mul_quantize": ([_p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_unpack_allspark": ([_p, _p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_quantize_block32": ([_p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_q8_block_mm": ([_p, _p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_q8_block_int8": ([_p, _p, _p, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_gguf_q8_packed_mm": ([_p, _p, _p, _p, _i64, _i64, _i64, _i64, _i64, _i64, _p],
                              ctypes.c_int),
}

# include/consumer_int8_attention.h: descriptors are passed by address.


class Heads(ctypes.Structure):
    _fields_ = [("data", _p), ("heads", _i64), ("token_stride", _i64), ("head_stride", _i64)]


class HeadNorm(ctypes.Structure):
    _fields_ = [("q_weight", _p), ("k_weight", _p), ("eps", ctypes.c_double)]


class Rotation(ctypes.Structure):
    _fields_ = [("table", _p), ("rows", _i64), ("rot", _i64), ("positions", _p), ("axes", _i64),
                ("axis_of", _p), ("interleaved", _i64)]


class Fp4CacheView(ctypes.Structure):
    _fields_ = [("k_codes", _p), ("k_scales", _p), ("v_codes", _p), ("v_scales", _p),
                ("k_code_page_stride", _i64), ("k_scale_page_stride", _i64),
                ("v_code_page_stride", _i64), ("v_scale_page_stride", _i64), ("pages", _i64),
                ("heads", _i64), ("page_size", _i64)]


_heads, _norm, _rotation, _cache = (ctypes.POINTER(t)
                                    for t in (Heads, HeadNorm, Rotation, Fp4CacheView))

ATTENTION_SIGNATURES = {
    "ci8_qk_norm_rope": ([_heads, _heads, _heads, _heads, _norm, _rotation, _i64, _i64, _p],
                         ctypes.c_int),
    "ci8_append_fp4": ([_heads, _heads, _heads, _heads, _norm, _rotation, _p, _cache, _i64, _i64,
                        _p], ctypes.c_int),
    "ci8_unpack_fp4": ([_cache, _p, _p, _p, _i64, _i64, _p], ctypes.c_int),
    "ci8_attention_fp4": ([_heads, _cache, _p, _i64, _p, _p, _i64, _i64, _i64, _p, _p, _p,
                           ctypes.c_double, _i64, _i64, _p], ctypes.c_int),
}

# include/consumer_int8_drafts.h
DRAFTS_SIGNATURES = {
    "ci8_attention_fp4_tree": ([_heads, _cache, _p, _i64, _p, _p, _p, _i64, _i64, _i64, _p, _p, _p,
                                ctypes.c_double, _i64, _i64, _p], ctypes.c_int),
    "ci8_move_fp4": ([_cache, _p, _p, _p, _i64, _i64, _i64, _p], ctypes.c_int),
    "ci8_token_probs": ([_p, _i64, _i64, _p, _p, _i64, _i64, _i64, _p, _p], ctypes.c_int),
    "ci8_verify_drafts": ([_p, _i64, _p, _i64, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p, _p, _p, _p],
                          ctypes.c_int),
}

_lib = None


def load(path: Path | str = LIB_PATH) -> ctypes.CDLL:
    global _lib
    if _lib is None:
        lib = ctypes.CDLL(str(path))
        for name, (args, res) in {**SIGNATURES, **ATTENTION_SIGNATURES,
                                      **DRAFTS_SIGNATURES}.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = res
        _lib = lib
    return _lib


def last_error() -> str:
    return load().ci8_last_error().decode()


def check(status: int) -> None:
    if status != CI8_OK:
        raise RuntimeError(last_error())
