"""The operator boundary: ``alexdremov_cross_attention::{forward, backward}``, ``alexdremov_paged_attention::{forward, append, append_rope,
tree_forward, keep}`` and ``alexdremov_qk_norm_rope::{forward, backward}``.

The ops, their GPU implementation (which enqueues the HIP kernels of libkv_attention.so on the current stream) and their autograd are
native code (csrc/kv_torch.cpp, kv_rope_torch.cpp, module ``_native``); this file holds the fake implementations and the argument checks.
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


def _check_pages(k_pages, v_pages, page_table):
    assert k_pages.shape[2] >= 1, "a page holds at least one position"
    for t in (k_pages, v_pages):
        vec = 16 // t.element_size()
        ok = t.stride(3) == 1 and (t.device.type == "meta" or t.data_ptr() % 16 == 0)
        ok = ok and all(n <= 1 or (s > 0 and s % vec == 0) for n, s in zip(t.shape[:3], t.stride()))
        assert t.numel() == 0 or ok, \
            "pages are read and written in place: unit stride along the head dimension, others and the address multiples of 16 bytes"
    assert page_table.dtype == torch.int32 and page_table.ndim == 2, "page_table must be int32 of shape (batch, pages of a sequence)"
    assert page_table.device == k_pages.device, "page_table must be on the device of q"
    assert page_table.shape[1] * k_pages.shape[2] <= MOST_POSITIONS, "a sequence has at most 2**30 positions"


def _validate_cache(x, k_pages, v_pages, page_table, lens, new_lens):
    _check_heads(x, k_pages, v_pages)
    _check_pages(k_pages, v_pages, page_table)
    assert page_table.shape[0] == x.shape[0], "page_table must be int32 of shape (batch, pages of a sequence)"
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


def _validate_tree(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens):
    _validate_cache(q, k_pages, v_pages, page_table, lens, new_lens)
    T = q.shape[2]
    assert tree.dtype == torch.bool and tuple(tree.shape) in ((T, T), (q.shape[0], T, T)), \
        "tree must be bool of shape (tokens, tokens) or (batch, tokens, tokens)"
    assert tree.device == q.device, "tree must be on the device of q"
    _check_scale(sm_scale)


def _validate_keep(k_pages, v_pages, page_table, first, kept):
    assert k_pages.ndim == 4 and k_pages.dtype in DTYPES, f"unsupported cache {k_pages.dtype}: expected float32, float16 or bfloat16 pages"
    assert k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype and k_pages.device == v_pages.device, \
        "keys and values need one shape, type and device"
    assert k_pages.shape[-1] in HEAD_DIMS and k_pages.shape[1] >= 1
    _check_pages(k_pages, v_pages, page_table)
    B = page_table.shape[0]
    assert first.dtype == torch.int32 and tuple(first.shape) == (B,), "first must be int32 of shape (batch,)"
    assert kept.dtype == torch.int32 and kept.ndim == 2 and kept.shape[0] == B, "kept must be int32 of shape (batch, entries)"
    assert first.device == k_pages.device and kept.device == k_pages.device, "first and kept must be on the device of the pages"
    assert max(k_pages.shape) <= _INT32 and max(kept.shape) <= _INT32 and max(page_table.shape) <= _INT32


def _check_pair(q, k, lens):
    assert q.ndim == 4 and k.ndim == 4
    assert k.device == q.device, "queries and keys must be on one device"
    assert q.dtype == k.dtype
    assert q.dtype in DTYPES, f"unsupported dtype {q.dtype}: expected float32, float16 or bfloat16"
    assert q.shape[-1] in HEAD_DIMS
    assert (k.shape[0], k.shape[2], k.shape[3]) == (q.shape[0], q.shape[2], q.shape[3]), "queries and keys need one batch, tokens and head dimension"
    assert q.shape[1] >= 1 and k.shape[1] >= 1
    assert max(q.shape) <= _INT32 and max(k.shape) <= _INT32
    _check_lengths("lens", lens, q)


def _check_rotation(q, cos, sin, q_weight, k_weight, positions, eps):
    for t in (cos, sin):
        assert t.dtype == torch.float32 and t.ndim == 2, "cos and sin must be float32 of shape (positions, rotated channels / 2)"
        assert t.device == q.device, "cos and sin must be on the device of q"
    assert cos.shape == sin.shape, "cos and sin need one shape"
    rot = 2 * cos.shape[1]
    assert 16 <= rot <= q.shape[-1] and rot % 16 == 0, "the rotated channels must be a multiple of 16, up to the head dimension"
    assert cos.shape[0] <= _INT32
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        assert w is None or (tuple(w.shape) == (q.shape[-1],) and w.dtype in (q.dtype, torch.float32)), \
            f"{name} must be of shape (head_dim,), in q's type or float32"
        assert w is None or w.device == q.device, f"{name} must be on the device of q"
    assert q_weight is None or k_weight is None or q_weight.dtype == k_weight.dtype, "q_weight and k_weight need one type"
    assert positions is None or (positions.dtype == torch.int32 and tuple(positions.shape) == (q.shape[0], q.shape[2])), \
        "positions must be int32 of shape (batch, tokens)"
    assert positions is None or positions.device == q.device, "positions must be on the device of q"
    assert eps is not None or (q_weight is None and k_weight is None), "weights are those of the norms: give eps too"
    assert eps is None or (math.isfinite(eps) and 2.0 ** -149 < eps < 3.4e38), "eps must be a positive number of float32"


def _validate_rope(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, *grads):
    """Called by the native implementation with arguments it cannot serve, to name the condition."""
    _check_pair(q, k, lens)
    _check_rotation(q, cos, sin, q_weight, k_weight, positions, eps)
    for g, x in zip(grads, (q, k)):
        assert g.shape == x.shape, "gradients need the shapes of q and k"
        assert g.device == x.device, "gradients must be on the device of q"


def _validate_append_rope(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps):
    _validate_cache(q, k_pages, v_pages, page_table, lens, new_lens)
    _check_pair(q, k, None)
    assert k.shape == v.shape and k.dtype == v.dtype and k.device == v.device, "k and v need one shape, type and device"
    assert k.shape[1] == k_pages.shape[1], "k and v need the heads of the pages"
    _check_rotation(q, cos, sin, q_weight, k_weight, positions, eps)


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


@torch.library.register_fake("alexdremov_paged_attention::tree_forward")
def _tree_forward_abstract(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse):
    return torch.empty_like(q, memory_format=torch.contiguous_format), _rows(q, return_lse)


@torch.library.register_fake("alexdremov_paged_attention::keep")
def _paged_keep_abstract(k_pages, v_pages, page_table, first, kept):
    return None


@torch.library.register_fake("alexdremov_paged_attention::append_rope")
def _append_rope_abstract(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps, interleaved):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


@torch.library.register_fake("alexdremov_qk_norm_rope::forward")
def _rope_forward_abstract(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k))


@torch.library.register_fake("alexdremov_qk_norm_rope::backward")
def _rope_backward_abstract(d_q, d_k, q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved, weights):
    rows = tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k))
    return rows + tuple(torch.empty(0, dtype=q.dtype, device=q.device) if w is None or not weights else
                        torch.empty(w.shape, dtype=w.dtype, device=w.device) for w in (q_weight, k_weight))


_torch_function_modes = torch._C._len_torch_function_stack
_is_compiling = torch.compiler.is_compiling
_PLAIN = {torch.Tensor, type(None)}


def takes_native_call(*tensors) -> bool:
    """Plain tensors with no torch-function mode around go from Python to the dispatcher in one native call; subclasses,
    proxies and modes need the Python op call, which they can intercept."""
    return not _is_compiling() and _PLAIN.issuperset(map(type, tensors)) and not _torch_function_modes()
