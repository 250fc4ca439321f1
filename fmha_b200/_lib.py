"""ctypes binding of libfmha_b200.so (the C ABI declared in include/fmha.h).

Loading fails loudly: there is no CPU or PyTorch fallback for any entry point.
"""
from __future__ import annotations

import ctypes
import os

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libfmha_b200.so")

FMHA_OK = 0
FMHA_ERR_INVALID_ARG = 1
FMHA_ERR_UNSUPPORTED = 2
FMHA_ERR_MISALIGNED = 3
FMHA_ERR_CUDA = 4
FMHA_ERR_DEVICE_TIMEOUT = 5

VARIANT_AUTO, VARIANT_BULK, VARIANT_LDG = 0, 1, 2
DTYPE_BF16, DTYPE_FP16, DTYPE_E4M3 = 0, 1, 2
VARIANTS = {"auto": VARIANT_AUTO, "bulk": VARIANT_BULK, "ldg": VARIANT_LDG}

_vp, _i, _i64, _u64, _u32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_uint32
_f = ctypes.c_float


class PagedCacheStruct(ctypes.Structure):
    """fmha_paged_cache_t (include/fmha.h)."""
    _fields_ = [("k", _vp), ("v", _vp), ("block_table", _vp), ("seqlens_kv", _vp),
                ("page_stride", _i64), ("head_stride", _i64), ("token_stride", _i64),
                ("table_stride", _i64), ("num_pages", _i), ("page_size", _i), ("max_pages", _i),
                ("dtype", _i), ("k_scale", _f), ("v_scale", _f)]


class RopeAppendArgs(ctypes.Structure):
    """fmha_rope_append_args_t."""
    _fields_ = [(n, _vp) for n in ("q", "k", "v", "q_out", "k_out", "cu_seqlens_q", "cos_table",
                                   "sin_table")] + \
               [(n, _i64) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride",
                                    "k_out_stride")] + [("cache", PagedCacheStruct)] + \
               [(n, _i) for n in ("total_tokens", "batch", "num_heads_q", "num_heads_kv",
                                  "head_dim", "rotary_dim", "max_position", "interleaved", "dtype")]


class PagedDecodeArgs(ctypes.Structure):
    """fmha_paged_decode_args_t."""
    _fields_ = [(n, _vp) for n in ("q", "o", "lse", "workspace")] + \
               [(n, _i64) for n in ("workspace_bytes", "q_stride", "o_stride")] + \
               [("cache", PagedCacheStruct)] + \
               [(n, _i) for n in ("batch", "num_heads_q", "num_heads_kv", "head_dim", "dtype",
                                  "o_dtype")] + [("softmax_scale", _f)]


class PromptArgs(ctypes.Structure):
    """fmha_prompt_args_t."""
    _fields_ = [(n, _vp) for n in ("q", "k", "v", "o", "lse", "cu_seqlens_q", "cu_seqlens_kv")] + \
               [(n, _i64) for n in ("q_stride", "k_stride", "v_stride", "o_stride")] + \
               [(n, _i) for n in ("total_q", "total_kv", "batch", "num_heads_q", "num_heads_kv",
                                  "head_dim", "causal", "dtype", "o_dtype")] + \
               [("softmax_scale", _f)]


# Every symbol include/fmha.h declares, with (restype, argtypes).
SIGNATURES = {
    "fmha_forward": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "fmha_forward_variant": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "fmha_forward_noalloc": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "fmha_forward_varlen": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, ctypes.c_float, _vp]),
    "fmha_forward_varlen_variant": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i,
                                         ctypes.c_float, _i, _vp]),
    "fmha_forward_append": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "fmha_rope_append": (_i, [_vp, _vp]),
    "fmha_paged_decode_workspace": (_i64, [_i, _i, _i, _i64]),
    "fmha_paged_decode": (_i, [_vp, _vp]),
    "fmha_prompt": (_i, [_vp, _vp]),
    "fmha_status_string": (ctypes.c_char_p, [_i]),
    "fmha_device_error": (_i, [ctypes.POINTER(_i)]),
    "fmha_fill_normal_bf16": (_i, [_vp, _i64, _u64, _u32, _i64, _vp]),
    "fmha_version": (ctypes.c_char_p, []),
    "fmha_seqlens_poisson": (_i, [_i, _i, _u32, ctypes.c_double, _vp]),
    "fmha_test_inject_stall": (None, [_i]),
}

_lib = None


class FmhaError(RuntimeError):
    def __init__(self, status: int, what: str = ""):
        self.status = status
        msg = status_string(status) if _lib is not None else f"status {status}"
        super().__init__(f"{what}: {msg}" if what else msg)


def load(path: str | None = None) -> ctypes.CDLL:
    """Loads the CUDA library (built in-tree by fmha_b200.build)."""
    global _lib
    if _lib is not None:
        return _lib
    path = path or LIB_PATH
    if not os.path.exists(path):
        raise ImportError(
            f"{path} is missing: build it with `python -m fmha_b200.build` "
            "(fmha_b200 has no fallback implementation)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    _lib = lib
    return lib


def status_string(status: int) -> str:
    return load().fmha_status_string(int(status)).decode()


def check(status: int, what: str = "") -> None:
    if status != FMHA_OK:
        raise FmhaError(status, what)
