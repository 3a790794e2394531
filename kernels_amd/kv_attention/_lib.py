"""ctypes binding of libkv_attention.so (the C ABI in include/kv_attention.h).

The library is the only compute path: if it cannot be loaded the operators raise, they never fall back to a PyTorch
implementation.
"""
from __future__ import annotations

import ctypes
import os
import threading

_LIB_NAME = "libkv_attention.so"
_lock = threading.Lock()
_lib = None

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_st = ctypes.POINTER(ctypes.c_int64)
_lengths = [_vp, _i64]

# name -> argument types, in the order of include/kv_attention.h
SIGNATURES = {
    "kv_cross_forward_workspace": [_i32] * 7,
    "kv_cross_forward": [_vp] * 3 + _lengths * 2 + [_vp, _vp, _vp, _i64] + [_st] * 3 + [_i32] * 6 + [_f32, _i32, _vp],
    "kv_cross_backward_workspace": [_i32] * 7,
    "kv_cross_backward": [_vp] * 3 + _lengths * 2 + [_vp] * 6 + [_vp, _i64] + [_st] * 5 + [_i32] * 6 + [_f32, _i32, _vp],
    "kv_paged_forward_workspace": [_i32] * 10,
    "kv_paged_forward": [_vp] * 3 + _lengths * 3 + [_vp, _vp, _vp, _i64] + [_st] * 3 + [_i32] * 10 + [_f32, _i32, _vp],
    "kv_paged_append": [_vp] * 4 + _lengths * 3 + [_st] * 4 + [_i32] * 8 + [_vp],
    "kv_paged_tree_forward_workspace": [_i32] * 8,
    "kv_paged_tree_forward": [_vp] * 3 + _lengths * 3 + [_vp, _st] + [_vp, _vp, _vp, _i64] + [_st] * 3 + [_i32] * 8 + [_f32, _i32, _vp],
    "kv_paged_keep": [_vp] * 2 + _lengths * 2 + [_vp, _st] + [_st] * 2 + [_i32] * 8 + [_vp],
    "kv_qk_norm_rope": [_vp] * 4 + [_i64] * 2 + [_vp] * 2 + [_i32] + _lengths + [_vp, _st] + [_vp] * 2 + [_st] * 2 + [_i32] * 8 + [_f32, _i32, _vp],
    "kv_qk_norm_rope_backward_workspace": [_i32] * 6,
    "kv_qk_norm_rope_backward": [_vp] * 6 + [_i64] * 2 + [_vp] * 2 + [_i32] + _lengths + [_vp, _st] + [_vp] * 5 + [_i64] + [_st] * 4 + [_i32] * 8
                                + [_f32, _i32, _vp],
    "kv_paged_append_rope": [_vp] * 6 + _lengths * 3 + [_vp] * 2 + [_i64] * 2 + [_vp] * 2 + [_i32] + [_vp, _st] + [_st] * 5 + [_i32] * 11
                            + [_f32, _i32, _vp],
    "kv_error_string": [_i32],
}


def library_path() -> str:
    return os.environ.get("KV_ATTENTION_LIB", os.path.join(os.path.dirname(os.path.abspath(__file__)), _LIB_NAME))


def load() -> ctypes.CDLL:
    """Load the shared library once and attach argument types to its entry points."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not os.path.exists(path):
            raise RuntimeError(
                f"{_LIB_NAME} not found at {path}: build it with `make -C kernels_amd/csrc` "
                "(or `python -c 'import __graft_entry__ as g; g.build()'`). "
                "There is no fallback implementation."
            )
        lib = ctypes.CDLL(path)
        for name, argtypes in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = argtypes
            fn.restype = ctypes.c_char_p if name == "kv_error_string" else _i64 if name.endswith("_workspace") else _i32
        _lib = lib
    return _lib


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}: {load().kv_error_string(rc).decode()}")


def strides4(t) -> ctypes.Array:
    """The four element strides of ``t`` as an int64[4]; a dimension of one element counts as stride 0."""
    return (ctypes.c_int64 * 4)(*(st if n > 1 or i == 3 else 0 for i, (n, st) in enumerate(zip(t.shape, t.stride()))))
