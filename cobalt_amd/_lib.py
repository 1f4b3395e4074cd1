"""Bindings of libcbk_hip.so: ctypes for the C ABI declared in include/cbk.h, and the extension
module `_native` with the operators that are called per token.

The library is the only compute path of this package: if it is not built, every operator
raises instead of falling back to PyTorch."""
from __future__ import annotations

import ctypes
import os

from .format import CbkDesc  # noqa: F401 (re-exported for callers that build descriptor arrays)


class CbkCache(ctypes.Structure):
    """struct cbk_cache (include/cbk.h)"""
    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p), ("k_meta", ctypes.c_void_p),
                ("v_meta", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page", ctypes.c_int32), ("heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("group", ctypes.c_int32)]


class CbkRows(ctypes.Structure):
    """struct cbk_rows (include/cbk.h)"""
    _fields_ = [("table", ctypes.c_void_p), ("ld_table", ctypes.c_int64), ("lens", ctypes.c_void_p),
                ("starts", ctypes.c_void_p), ("seqs", ctypes.c_int32), ("table_cols", ctypes.c_int32),
                ("tokens", ctypes.c_int64)]


_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libcbk_hip.so")
_lib = None

_P = ctypes.c_void_p
_DP = ctypes.POINTER(CbkDesc)
_MM = [_DP, _P, ctypes.c_int, ctypes.c_int, ctypes.c_int64, _P, ctypes.c_int, ctypes.c_int64, _P, _P,
       ctypes.c_size_t, _P]
_CP, _RP = ctypes.POINTER(CbkCache), ctypes.POINTER(CbkRows)
_ROWS = [_P, ctypes.c_int64, ctypes.c_int64]                        # a dense tensor: address, strides of rows and heads
SIGNATURES = {
    "cbk_abi_version": (ctypes.c_int, []),
    "cbk_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "cbk_desc_check": (ctypes.c_int, [_DP, _DP]),
    "cbk_row_stride": (ctypes.c_size_t, [_DP]),
    "cbk_stream_bytes": (ctypes.c_size_t, [_DP, ctypes.c_size_t]),
    "cbk_workspace_bytes": (ctypes.c_size_t, [_DP, ctypes.c_int]),
    "cbk_pack": (ctypes.c_int, [_DP, _P, _P, _P, _P, ctypes.c_int, ctypes.c_int, _P, _P]),
    "cbk_unpack": (ctypes.c_int, [_DP, _P, _P, _P]),
    "cbk_dequant": (ctypes.c_int, [_DP, ctypes.c_int, ctypes.c_int, ctypes.c_int, _P, ctypes.c_int,
                                   ctypes.c_int64, _P]),
    "cbk_gemv": (ctypes.c_int, _MM),
    "cbk_gemm": (ctypes.c_int, _MM),
    "cbk_gemm_static": (ctypes.c_int, _MM[:9] + [_P]),
    "cbk_gemv_batch_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, _DP, ctypes.c_int]),
    "cbk_gemv_batch": (ctypes.c_int, [ctypes.c_int, _DP, ctypes.POINTER(_P), ctypes.POINTER(ctypes.c_int64),
                                      ctypes.c_int, ctypes.c_int, ctypes.POINTER(_P), ctypes.POINTER(ctypes.c_int64),
                                      ctypes.c_int, ctypes.POINTER(_P), _P, ctypes.c_size_t, _P]),
    "cbk_linear": (ctypes.c_int, _MM),
    "cbk_linear_act_workspace_bytes": (ctypes.c_size_t, [_DP, ctypes.c_int, ctypes.c_int]),
    "cbk_linear_act": (ctypes.c_int, _MM[:9] + [ctypes.c_int] + _MM[9:]),
    "cbk_cache_code_bytes": (ctypes.c_size_t, [_CP]),
    "cbk_cache_meta_bytes": (ctypes.c_size_t, [_CP]),
    "cbk_cache_write": (ctypes.c_int, [_CP, _RP] + _ROWS + _ROWS + [ctypes.c_int, _P]),
    "cbk_cache_read": (ctypes.c_int, [_CP, _RP] + _ROWS + _ROWS + [ctypes.c_int, _P]),
    "cbk_cache_attention_workspace_bytes": (ctypes.c_size_t, [_CP, _RP, ctypes.c_int]),
    "cbk_cache_attention": (ctypes.c_int, [_CP, _RP] + _ROWS + _ROWS + [ctypes.c_int, ctypes.c_int, ctypes.c_float, ctypes.c_int,
                                                                      ctypes.c_int, _P, ctypes.c_size_t, _P]),
}
ACT_CODE = {"gelu_tanh": 0, "silu": 1}


class CbkError(RuntimeError):
    pass


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise CbkError(f"{LIB_PATH} is missing: build it with `python -m cobalt_amd.build` "
                           "(hipcc, gfx950). There is no PyTorch fallback.")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        if L.cbk_abi_version() != 1:
            raise CbkError(f"ABI version {L.cbk_abi_version()} != 1")
        _lib = L
    return _lib


_native = None


def native():
    """The extension module with the operators (`_native.so`); raises if it has not been built."""
    global _native
    if _native is None:
        lib()
        try:
            from . import _native as mod
        except ImportError as e:
            raise CbkError("cobalt_amd/_native.so is missing or does not load: build it with "
                           f"`python -m cobalt_amd.build`. There is no PyTorch fallback. ({e})") from e
        mod.set_error(CbkError)
        _native = mod
    return _native


def check(rc: int, what: str):
    if rc != 0:
        raise CbkError(f"{what} failed: {lib().cbk_strerror(rc).decode()} (status {rc})")
