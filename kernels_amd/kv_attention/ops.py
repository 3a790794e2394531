"""The operator boundary: ``alexdremov_cross_attention::{forward, backward}`` and ``alexdremov_paged_attention::{forward, append}``.

The ops, their GPU implementation (which enqueues the HIP kernels of libkv_attention.so on the current stream) and their autograd are
native code (csrc/kv_torch.cpp, module ``_native``); this file holds the fake implementations and the argument checks.
"""
from __future__ import annotations

import math

import torch

try:
    from . import _native  # noqa: F401  (the module registers the ops)
except ImportError as e:
    raise ImportError(
        "kv_attention._native cannot be loaded: build it with `make -C kernels_amd/csrc` "
        "(or `python -c 'import __graft_entry__ as g; g.build()'`). There is no fallback implementation."
    ) from e

HEAD_DIMS = (16, 32, 64, 128, 256)
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MOST_POSITIONS = 1 << 30   # page_table.shape[1] * page size
MOST_SCALE = 2.0 ** 127    # the kernels take it times log2(e), in float32
_INT32 = 2 ** 31 - 1


def _check_lengths(name, lens, q):
    assert lens is None or (lens.dtype == torch.int32 and lens.ndim == 1 and len(lens) == q.shape[0]), \
        f"{name} must be int32 of shape (batch,)"
    assert lens is None or lens.device == q.device, f"{name} must be on the device of q"


def _check_scale(sm_scale):
    assert math.isfinite(sm_scale), "sm_scale must be finite"
    assert abs(sm_scale) <= MOST_SCALE, "sm_scale must lie within 2**127 on either side of 0"


def _check_heads(q, k, v):
    assert q.ndim == 4 and k.ndim == 4 and v.ndim == 4
    assert k.device == q.device and v.device == q.device, "queries, keys and values must be on one device"
    assert q.dtype == k.dtype == v.dtype
    assert q.dtype in DTYPES, f"unsupported dtype {q.dtype}: expected float32, float16 or bfloat16"
    assert k.shape == v.shape, "keys and values need one shape"
    assert q.shape[-1] in HEAD_DIMS
    assert k.shape[-1] == q.shape[-1]
    assert k.shape[1] >= 1 and q.shape[1] >= 1 and q.shape[1] % k.shape[1] == 0, \
        "the query heads must be a multiple of the key heads"
    assert max(q.shape) <= _INT32 and max(k.shape) <= _INT32


def _validate_cross(q, k, v, lens, q_lens, sm_scale, *others):
    """Called by the native implementation with arguments it cannot serve, to name the condition."""
    _check_heads(q, k, v)
    assert k.shape[0] == q.shape[0], "k and v need q's batch size"
    _check_lengths("lens", lens, q)
    _check_lengths("q_lens", q_lens, q)
    _check_scale(sm_scale)
    for t in others:
        assert t.shape == q.shape, "o and dO need q's shape"
        assert t.device == q.device, "o and dO must be on the device of q"


def _validate_cache(x, k_pages, v_pages, page_table, lens, new_lens):
    _check_heads(x, k_pages, v_pages)
    assert k_pages.shape[2] >= 1, "a page holds at least one position"
    for t in (k_pages, v_pages):
        vec = 16 // t.element_size()
        ok = t.stride(3) == 1 and (t.device.type == "meta" or t.data_ptr() % 16 == 0)
        ok = ok and all(n <= 1 or (s > 0 and s % vec == 0) for n, s in zip(t.shape[:3], t.stride()))
        assert t.numel() == 0 or ok, \
            "pages are read and written in place: unit stride along the head dimension, others and the address multiples of 16 bytes"
    assert page_table.dtype == torch.int32 and page_table.ndim == 2 and page_table.shape[0] == x.shape[0], \
        "page_table must be int32 of shape (batch, pages of a sequence)"
    assert page_table.device == x.device, "page_table must be on the device of q"
    assert page_table.shape[1] * k_pages.shape[2] <= MOST_POSITIONS, "a sequence has at most 2**30 positions"
    assert lens is not None
    _check_lengths("lens", lens, x)
    _check_lengths("new_lens", new_lens, x)


def _validate_paged(q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale, new_lens):
    _validate_cache(q, k_pages, v_pages, page_table, lens, new_lens)
    assert back_contexts >= 0 and context_size >= 1
    _check_scale(sm_scale)


def _validate_append(k, v, k_pages, v_pages, page_table, lens, new_lens):
    _validate_cache(k, k_pages, v_pages, page_table, lens, new_lens)
    assert k.shape == v.shape and k.dtype == v.dtype and k.device == v.device, "k and v need one shape, type and device"
    assert k.shape[1] == k_pages.shape[1], "k and v need the heads of the pages"


def _rows(q, return_lse):
    return torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else torch.empty(0)


@torch.library.register_fake("alexdremov_cross_attention::forward")
def _cross_forward_abstract(q, k, v, lens, q_lens, sm_scale, return_lse):
    return torch.empty_like(q, memory_format=torch.contiguous_format), _rows(q, return_lse)


@torch.library.register_fake("alexdremov_cross_attention::backward")
def _cross_backward_abstract(q, k, v, lens, q_lens, o, lse, do, sm_scale):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))


@torch.library.register_fake("alexdremov_paged_attention::forward")
def _paged_forward_abstract(q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale, new_lens, return_lse):
    return torch.empty_like(q, memory_format=torch.contiguous_format), _rows(q, return_lse)


@torch.library.register_fake("alexdremov_paged_attention::append")
def _paged_append_abstract(k, v, k_pages, v_pages, page_table, lens, new_lens):
    return None


_torch_function_modes = torch._C._len_torch_function_stack
_is_compiling = torch.compiler.is_compiling
_PLAIN = {torch.Tensor, type(None)}


def takes_native_call(*tensors) -> bool:
    """Plain tensors with no torch-function mode around go from Python to the dispatcher in one native call; subclasses,
    proxies and modes need the Python op call, which they can intercept."""
    return not _is_compiling() and _PLAIN.issuperset(map(type, tensors)) and not _torch_function_modes()
