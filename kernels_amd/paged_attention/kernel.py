"""``paged_attention``, ``paged_tree_attention``, ``paged_append``, ``paged_append_rope`` and ``paged_keep`` over the
``alexdremov_paged_attention`` ops (kernels: csrc/kv_rows.h, kv_append.h, kv_rope.h)."""
from __future__ import annotations

import torch

from kv_attention import ops
from kv_attention._native import paged_append as _eager_append
from kv_attention._native import paged_append_rope as _eager_append_rope
from kv_attention._native import paged_attention as _eager_call
from kv_attention._native import paged_keep as _eager_keep
from kv_attention._native import paged_tree_attention as _eager_tree

_NO_LIMIT = 2 ** 31 - 1


def paged_attention_reference(q, k_pages, v_pages, page_table, lens, context_size=1, back_contexts=None, sm_scale=None, new_lens=None):
    """The same in plain PyTorch, in the inputs' type; returns ``(output, valid_token_mask)``.  Meant for checking, not for use."""
    B, Hq, T, D = q.shape
    N, Hkv, page, _ = k_pages.shape
    width, dev = page_table.shape[1], q.device
    lens = lens.to(dev).long().clamp(0, width * page)[:, None]
    count = torch.full_like(lens, T) if new_lens is None else new_lens.to(dev).long().clamp(0, T)[:, None]
    at = torch.arange(width * page, device=dev)
    there = ((page_table >= 0) & (page_table < N)).repeat_interleave(page, dim=1)
    pages = page_table.long().clamp(0, max(N - 1, 0))
    k, v = (x[pages].transpose(1, 2).reshape(B, Hkv, width * page, D) for x in (k_pages, v_pages))
    i = torch.arange(T, device=dev)
    where = lens - count + i                                        # positions of the new tokens
    gap = torch.div(where, context_size, rounding_mode="floor")[:, :, None] - torch.div(at, context_size, rounding_mode="floor")
    seen = (gap >= 0) & (at < lens)[:, None] & (where >= 0)[:, :, None] & there[:, None]
    if back_contexts is not None:
        seen &= gap <= back_contexts
    v = torch.where(seen.any(1)[:, None, :, None], v, 0.0)
    k, v = (x.repeat_interleave(Hq // Hkv, dim=1) for x in (k, v))
    scores = (q @ k.transpose(-1, -2)) * (D ** -0.5 if sm_scale is None else sm_scale)
    scores = scores.masked_fill(~seen[:, None], float("-inf"))
    some = seen.any(-1)[:, None, :, None]
    p = torch.softmax(torch.where(some, scores, 0.0), dim=-1) if scores.shape[-1] > 0 else scores
    valid = (i < count)[:, None, :, None]
    return torch.where(valid & some, p @ v, 0.0), valid


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    context_size: int = 1,
    back_contexts: int | None = None,
    sm_scale: float | None = None,
    new_lens: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """The newest tokens of every sequence over its cache: what :func:`streaming_attention.streaming_attention` gives for its
    last rows, from keys and values in pages.

    Args:
        q: ``(batch, heads, tokens, head_dim)``, the queries of the newest tokens; one token per sequence in a decoding step, a chunk
            of them in streaming
        k_pages, v_pages: ``(pages, key_heads, page_size, head_dim)``, read in place: unit stride along the head dimension, the
            others multiples of 16 bytes (a ``(pages, page_size, key_heads, head_dim)`` cache is passed transposed).  ``heads`` is a multiple of
            ``key_heads``; any page size
        page_table: ``(batch, width)`` int32.  Position ``t`` of sequence ``b`` is position ``t % page_size`` of page
            ``page_table[b, t // page_size]``.  An entry outside ``[0, pages)`` is a page that is not there: its positions are not seen
            (``-1`` for pages not yet taken, or given back when a window has left them)
        lens: ``(batch,)`` int32 lengths, the new tokens counted (:func:`paged_append` comes first); longer ones than the table holds
            count as what it holds
        context_size, back_contexts: a token at position ``t`` sees the positions ``j`` below ``lens[b]`` with
            ``0 <= t // context_size - j // context_size <= back_contexts``.  The default is causal attention to everything before;
            ``context_size=1, back_contexts=w`` is a window of ``w + 1`` positions
        sm_scale: softmax scale, ``head_dim ** -0.5`` by default
        new_lens: ``(batch,)`` int32 numbers of new tokens, or None for all of ``tokens``.  Token ``i`` of the ``n`` new ones of a sequence
            is at position ``lens[b] - n + i``
        return_lse: also return the base-2 log-sum-exp of the scaled scores, ``(batch, heads, tokens)`` float32

    Tokens beyond ``new_lens[b]`` give 0 and log-sum-exp 0; a token that sees no position gives 0 and log-sum-exp -inf.  What the cache holds
    where no token sees it does not matter.  (A value that is not finite, seen by one of several new tokens, reaches the others of
    its sequence.)  The bits of a sequence's result depend on the sizes of the call (the batch, the tokens, the table's width), not on the lengths or
    values of other sequences.  Forward only.  Can be captured into a HIP graph after one call of the same sizes and type outside the capture.

    Meant for few new tokens, in a table about as wide as its sequences are long: the work is divided by the table's width, and one or a few
    sequences of a table many times wider take several times as long as in a narrow one.  Prompts and further turns are served in any number
    of tokens and any head layout, at about a third of the rate of a large matrix product; a prompt of a sequence of its own, with as many key heads
    as heads, runs faster through :func:`streaming_attention.streaming_attention`, beside a :func:`paged_append`.
    """
    if back_contexts is None:
        back_contexts = _NO_LIMIT
    if ops.takes_native_call(q, k_pages, v_pages, page_table, lens, new_lens):
        result = _eager_call(q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale, new_lens, return_lse)
        if result is not NotImplemented:
            return result
    if sm_scale is None:
        sm_scale = q.size(-1) ** -0.5
    out, lse = torch.ops.alexdremov_paged_attention.forward(
        q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale, new_lens, return_lse)
    return (out, lse) if return_lse else out


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    new_lens: torch.Tensor | None = None,
) -> None:
    """Writes the keys and values of new tokens, ``(batch, key_heads, tokens, head_dim)``, into the pages, in place.

    ``lens[b]`` counts the new tokens already: token ``i`` of the ``n = new_lens[b]`` (or all) new ones goes to position ``lens[b] - n + i``.
    Positions below 0 or past the table, and pages that are not there, are left out; everything else in the cache stays
    as it is.  A page that sequences share (a common prefix) must not be written by more than one of them in a call: which of two values
    for one place stays is not defined; nor is what is written from ``k`` and ``v`` that overlap the pages.  Records no gradient: call it under
    ``torch.no_grad()`` or on detached tensors.
    """
    if ops.takes_native_call(k, v, k_pages, v_pages, page_table, lens, new_lens):
        if _eager_append(k, v, k_pages, v_pages, page_table, lens, new_lens) is not NotImplemented:
            return
    torch.ops.alexdremov_paged_attention.append(k, v, k_pages, v_pages, page_table, lens, new_lens)


def paged_append_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    new_lens: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    eps: float | None = None,
    interleaved: bool = False,
):
    """:func:`paged_append` with what :func:`qk_norm_rope.qk_norm_rope` does on the way: one pass from a projection's output to the cache.

    The keys of new tokens are turned by their positions, and with ``eps`` normed for each head first, as they go into the pages, the values
    go as they are, bit by bit, and the queries, ``(batch, heads, tokens, head_dim)``, come back turned likewise, ready for :func:`paged_attention` or
    :func:`paged_tree_attention`.

    Args:
        q, k, v, k_pages, v_pages, page_table, lens, new_lens: as for :func:`paged_append` and :func:`paged_attention`; the pages
            of keys and values, and what goes into them, must not overlap
        cos, sin, q_weight, k_weight, eps, interleaved: as for :func:`qk_norm_rope.qk_norm_rope`; no norms by default
        positions: ``(batch, tokens)`` int32 positions of the angles, or None: where the token goes, ``lens[b] - n + i``.  Drafted tokens of a tree
            stand behind each other in the cache, but each at the position of its depth

    Returns the queries; those of tokens beyond ``new_lens[b]`` are 0.  A token at a position that ``cos`` and ``sin`` do not have is left out of the
    cache and its queries are 0.  Records no gradient: call it under ``torch.no_grad()`` or on detached tensors.
    """
    if ops.takes_native_call(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions):
        result = _eager_append_rope(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps, interleaved)
        if result is not NotImplemented:
            return result
    return torch.ops.alexdremov_paged_attention.append_rope(
        q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps, interleaved)


def paged_tree_attention_reference(q, k_pages, v_pages, page_table, lens, tree, sm_scale=None, new_lens=None):
    """The same in plain PyTorch, in the inputs' type; returns ``(output, valid_token_mask)``.  Meant for checking, not for use."""
    B, Hq, T, D = q.shape
    N, Hkv, page, _ = k_pages.shape
    span, dev = page_table.shape[1] * page, q.device
    lens = lens.to(dev).long().clamp(0, span)[:, None]
    count = torch.full_like(lens, T) if new_lens is None else new_lens.to(dev).long().clamp(0, T)[:, None]
    at, i = torch.arange(span, device=dev), torch.arange(T, device=dev)
    there = ((page_table >= 0) & (page_table < N)).repeat_interleave(page, dim=1)
    pages = page_table.long().clamp(0, max(N - 1, 0))
    k, v = (x[pages].transpose(1, 2).reshape(B, Hkv, span, D) for x in (k_pages, v_pages))
    first = lens - count
    new = at - first                                                  # which of the new tokens a position holds
    drafted = tree.to(dev).expand(B, T, T).gather(2, new.clamp(0, max(T - 1, 0))[:, None].expand(B, T, span)) if T > 0 else there[:, None]
    seen = (new < 0)[:, None] | (drafted & (new >= 0)[:, None])
    seen = seen & ((at < lens) & there)[:, None] & ((first + i) >= 0)[:, :, None] & (i < count)[:, :, None]
    v = torch.where(seen.any(1)[:, None, :, None], v, 0.0)
    k, v = (x.repeat_interleave(Hq // Hkv, dim=1) for x in (k, v))
    scores = (q @ k.transpose(-1, -2)) * (D ** -0.5 if sm_scale is None else sm_scale)
    scores = scores.masked_fill(~seen[:, None], float("-inf"))
    some = seen.any(-1)[:, None, :, None]
    p = torch.softmax(torch.where(some, scores, 0.0), dim=-1) if span > 0 else scores
    return torch.where(some, p @ v, 0.0), (i < count)[:, None, :, None]


def paged_tree_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    tree: torch.Tensor,
    sm_scale: float | None = None,
    new_lens: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Attention of drafted tokens that form a tree (several continuations at once) over the cache, in one call.

    Args:
        q, k_pages, v_pages, page_table, lens, sm_scale, new_lens, return_lse: as for :func:`paged_attention`; the drafted tokens are the newest
            ones, in the cache already (:func:`paged_append_rope` with ``positions`` of their depths)
        tree: ``(tokens, tokens)`` bool, or ``(batch, tokens, tokens)``: ``tree[i, j]`` says that drafted token ``i`` sees drafted token ``j``: itself and
            its ancestors.  All see the positions before the drafted ones.  Any mask will do; entries of tokens beyond ``new_lens[b]`` are not used

    Token ``i`` of the ``n`` drafted ones is in the cache at position ``lens[b] - n + i``, whatever its depth; with the lower triangle as `tree`, this is
    :func:`paged_attention` with its default, causal windows.  There are no other windows (chunks, back contexts): every drafted token sees the whole
    context.  What that function says of padding, of tokens that see nothing, of values that are not finite, of bits, of capturing and of tables much wider
    than their sequences holds here too.  Forward only.  :func:`paged_keep` moves the accepted tokens together afterwards.
    """
    if ops.takes_native_call(q, k_pages, v_pages, page_table, lens, tree, new_lens):
        result = _eager_tree(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse)
        if result is not NotImplemented:
            return result
    if sm_scale is None:
        sm_scale = q.size(-1) ** -0.5
    out, lse = torch.ops.alexdremov_paged_attention.tree_forward(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse)
    return (out, lse) if return_lse else out


def paged_keep(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    first: torch.Tensor,
    kept: torch.Tensor,
) -> None:
    """Moves the keys and values of accepted tokens to the front of the drafted ones, in place.

    Args:
        k_pages, v_pages, page_table: the cache, as for :func:`paged_append`
        first: ``(batch,)`` int32 position of the first drafted token: the length before them
        kept: ``(batch, entries)`` int32: ``kept[b, i]`` is the drafted token that becomes the ``i``-th new one.  The path of a sequence ends at the
            first entry that is negative (-1 behind a shorter path) or not above the one before it: a token's ancestors stand before it

    ``first[b]`` and the number of kept tokens make the new length, which the caller counts.  Entries whose old or new place is not there (past the
    table, on a missing page) are left out; everything else in the cache stays as it is.  Pages that a call writes must stand
    in the table once, and the pages of keys and values must be the same or not overlap.  Records no gradient: call it under
    ``torch.no_grad()`` or on detached tensors.
    """
    if ops.takes_native_call(k_pages, v_pages, page_table, first, kept):
        if _eager_keep(k_pages, v_pages, page_table, first, kept) is not NotImplemented:
            return
    torch.ops.alexdremov_paged_attention.keep(k_pages, v_pages, page_table, first, kept)
