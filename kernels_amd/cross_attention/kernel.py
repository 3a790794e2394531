"""``cross_attention`` over the ``alexdremov_cross_attention`` ops (kernels: csrc/kv_fwd.h, kv_bwd.h, kv_rows.h)."""
from __future__ import annotations

import torch

from kv_attention import ops
from kv_attention._native import cross_attention as _eager_call


def cross_attention_reference(q, k, v, lens=None, q_lens=None, sm_scale=None):
    """The same in plain PyTorch, in the inputs' type; returns ``(output, valid_query_mask)``.  Meant for checking, not for use."""
    B, Hq, Tq, D = q.shape
    Tk, G = k.shape[2], Hq // k.shape[1]
    k, v = (t.repeat_interleave(G, dim=1) for t in (k, v))
    seen = torch.ones(B, Tk, dtype=torch.bool, device=q.device) if lens is None else \
        torch.arange(Tk, device=q.device) < lens.to(q.device)[:, None]
    valid = torch.ones(B, Tq, dtype=torch.bool, device=q.device) if q_lens is None else \
        torch.arange(Tq, device=q.device) < q_lens.to(q.device)[:, None]
    scores = (q @ k.transpose(-1, -2)) * (D ** -0.5 if sm_scale is None else sm_scale)
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    some = seen.any(-1)[:, None, None, None]
    p = torch.softmax(torch.where(some, scores, 0.0), dim=-1) if Tk > 0 else scores
    out = torch.where(some, p @ torch.where(seen[:, None, :, None], v, 0.0), 0.0)
    valid = valid[:, None, :, None]
    return torch.where(valid, out, 0.0), valid


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lens: torch.Tensor | None = None,
    q_lens: torch.Tensor | None = None,
    sm_scale: float | None = None,
    return_lse: bool = False,
):
    """Attention of every query to the first ``lens[b]`` keys, with gradients.

    Args:
        q: ``(batch, heads, queries, head_dim)``, float32 / float16 / bfloat16, head_dim 16, 32, 64, 128 or 256
        k, v: ``(batch, key_heads, keys, head_dim)``; ``heads`` is a multiple of ``key_heads``, and query head ``h`` reads key
            head ``h // (heads // key_heads)``
        lens: ``(batch,)`` int32 numbers of keys, or None
        q_lens: ``(batch,)`` int32 numbers of queries, or None
        sm_scale: softmax scale, ``head_dim ** -0.5`` by default
        return_lse: also return the base-2 log-sum-exp of the scaled scores, ``(batch, heads, queries)`` float32; no gradient
            flows through it

    Positions beyond a length are never used, whatever they hold.  Outputs and gradients there are 0 (and so is the log-sum-exp of
    a query beyond ``q_lens[b]``).  A query without a key has output 0 and log-sum-exp -inf and passes no gradient on.  Up to 32 queries of a
    key head (a decoding step) run a kernel that divides long runs of keys over the GPU.

    Results do not change from call to call.  Forward and backward can be captured into a HIP graph together, after one call
    of the same sizes and type outside the capture; as with any PyTorch operator, no graph of autograd that was recorded
    outside the capture and shares its leaves may be alive then.
    """
    if ops.takes_native_call(q, k, v, lens, q_lens):
        result = _eager_call(q, k, v, lens, q_lens, sm_scale, return_lse)
        if result is not NotImplemented:
            return result
    if sm_scale is None:
        sm_scale = q.size(-1) ** -0.5
    needs_lse = return_lse or (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)))
    out, lse = torch.ops.alexdremov_cross_attention.forward(q, k, v, lens, q_lens, sm_scale, needs_lse)
    return (out, lse) if return_lse else out
