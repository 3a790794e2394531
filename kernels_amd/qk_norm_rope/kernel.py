"""``qk_norm_rope`` over the ``alexdremov_qk_norm_rope`` ops (kernels: csrc/kv_rope.h)."""
from __future__ import annotations

import torch

from kv_attention import ops
from kv_attention._native import qk_norm_rope as _eager_call


def rotate_reference(x, cos, sin, weight=None, eps=None, interleaved=False):
    """One tensor ``(..., head_dim)`` with cosines and sines ``(..., rot / 2)`` that broadcast to it, in x's type."""
    rot = 2 * cos.shape[-1]
    if eps is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        x = x if weight is None else x * weight.to(x.dtype)
    cos, sin = cos.to(x.dtype), sin.to(x.dtype)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def qk_norm_rope_reference(q, k, cos, sin, q_weight=None, k_weight=None, lens=None, positions=None, eps=1e-6, interleaved=False):
    """The same in plain PyTorch, in the inputs' type.  Meant for checking, not for use."""
    B, _, T, _ = q.shape
    at = torch.arange(T, device=q.device).expand(B, T) if positions is None else positions.long()
    live = (at >= 0) & (at < cos.shape[0])
    if lens is not None:
        live &= torch.arange(T, device=q.device) < lens.to(q.device)[:, None]
    live = live[:, None, :, None]
    if cos.shape[0] > 0:
        rows = at.clamp(0, cos.shape[0] - 1)[:, None]
        cos, sin = cos[rows], sin[rows]
    else:
        cos, sin = cos.new_zeros(B, 1, T, cos.shape[1]), sin.new_zeros(B, 1, T, sin.shape[1])
    return tuple(torch.where(live, rotate_reference(torch.where(live, x, 1.0), cos, sin, w, eps, interleaved), 0.0)
                 for x, w in ((q, q_weight), (k, k_weight)))


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    lens: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    eps: float | None = 1e-6,
    interleaved: bool = False,
):
    """Queries and keys as attention takes them: each head's row over its root mean square, times the weights, and turned by its position.

    Args:
        q, k: ``(batch, heads, tokens, head_dim)`` and ``(batch, key_heads, tokens, head_dim)``, float32 / float16 / bfloat16, head_dim 16,
            32, 64, 128 or 256; views of a projection's output are read in place
        cos, sin: ``(positions, rot / 2)`` float32, the cosines and sines of every position's angles.  The first ``rot`` channels are turned, a
            multiple of 16 of them; the others stay as the norm leaves them
        q_weight, k_weight: ``(head_dim,)`` weights of the norms, in q's type or float32, or None (ones)
        lens: ``(batch,)`` int32 lengths, or None
        positions: ``(batch, tokens)`` int32 positions, or None: a token's place in its sequence
        eps: added to the mean square, or None: no norms (and no weights)
        interleaved: pairs are channels ``2 i`` and ``2 i + 1`` instead of ``i`` and ``i + rot / 2``

    Returns q and k, contiguous, in their type: ``(a cos - b sin, b cos + a sin)`` of every pair ``(a, b)`` of ``x * weight / sqrt(mean(x ** 2) + eps)``.
    Tokens beyond a length, and tokens at a position that the tables do not have, are padding: they give 0, are never used, whatever they
    hold, and pass no gradient on.  Gradients flow to q, k and the weights, not to the tables.  Sums are float32 (squares included: a row
    whose mean square float32 does not hold is out of range) and results are rounded once.

    Results do not change from call to call.  Forward and backward can be captured into a HIP graph together; as with any PyTorch operator, no
    graph of autograd that was recorded outside the capture and shares its leaves may be alive then.
    """
    if ops.takes_native_call(q, k, cos, sin, q_weight, k_weight, lens, positions):
        result = _eager_call(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved)
        if result is not NotImplemented:
            return result
    return torch.ops.alexdremov_qk_norm_rope.forward(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved)
