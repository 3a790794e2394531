"""float64 restatement of cross attention and of attention over pages, one (batch entry, query head) at a time, and bounds on what
the kernels' roundings may change, element by element.

The bounds count roundings (u: half a step of the element type, e: 2^-24 of float32) against sums of magnitudes:
  a score       e * (D + 4) * scale * |q| . |k|
  P             relative: twice the score's error (exp, and the sum it is divided by) + 2^-20 (exp2, log2) + u as an operand
  O             sum P |v| times P's relative error + u * |O| + e * (keys + 64) * sum P |v|
  delta         sum over D of O's error times |dO|
  dS            |dS| times P's relative error + P * (delta's error + e * (D + 4) * (sum |dO| |v| + sum |O| |dO|))
  dV, dQ, dK    the sums of those errors times the magnitudes they are multiplied with + u * |result| + the sums' own e
float16 operands below the smallest normal number are off by 2^-25 instead of u: P (of which a row's sum is at least 1 before the division) and dS.
"""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# results below the smallest normal number are rounded to its steps
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
E32 = 2.0 ** -24


def _head(q, k, v, seen, scale, dtype, g=None):
    """q [n, D], k, v [m, D], seen [n, m] in float64; returns results and bounds as {name: (value, bound)}."""
    u = 0.0 if dtype == torch.float32 else HALF_STEP[dtype]
    n, D = q.shape
    m = k.shape[0]
    live = seen.any(0)
    v = torch.where(live[:, None], v, 0.0)
    k = torch.where(live[:, None], k, 0.0)
    x = torch.where(seen, (q @ k.T) * scale, -math.inf)
    some = seen.any(-1)
    top = torch.where(some, x.amax(-1) if m else torch.zeros(n, dtype=q.dtype), 0.0)
    p = torch.exp(x - top[:, None])
    total = p.sum(-1)
    p = p / torch.where(total == 0, 1.0, total)[:, None]
    o = p @ v
    lse = torch.where(some, (top + torch.log(total)) / math.log(2), -math.inf)
    qk = abs(scale) * (q.abs() @ k.abs().T)
    ds_score = E32 * (D + 4) * qk
    worst = torch.where(seen, ds_score, 0.0).amax(-1, keepdim=True) if m else ds_score.sum(-1, keepdim=True)
    rel = 2 * worst + 2.0 ** -20   # of P in float32
    pv = p @ v.abs()
    final, tiny = HALF_STEP[dtype], TINY[dtype]
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    visible = seen.double()
    o_err = pv * (rel + u + E32 * (m + 64)) + final * o.abs() + tiny + sub * (visible @ v.abs())
    out = {"o": (o, o_err),
           "lse": (lse, torch.where(some, (worst[:, 0] * 2 + 2.0 ** -20 + E32 * (m + 64)) / math.log(2) + E32 * lse.abs() * 2, 0.0))}
    if g is None:
        return out
    dp = g @ v.T
    delta = (o * g).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    p_rel = rel + u + worst
    delta_err = (o_err * g.abs()).sum(-1, keepdim=True)
    sums = E32 * (D + 4) * (g.abs() @ v.abs().T + (o.abs() * g.abs()).sum(-1, keepdim=True))
    ds_err = ds.abs() * p_rel + p * (delta_err + sums)
    more = E32 * (max(m, n) + 64)
    dv = p.T @ g
    dq = scale * (ds @ k)
    dk = scale * (ds.T @ q)
    s = abs(scale)
    out["dv"] = (dv, (p * (p_rel + more) + sub * visible).T @ g.abs() + final * dv.abs() + tiny)
    out["dq"] = (dq, s * ((ds_err + ds.abs() * more + sub * visible) @ k.abs()) + final * dq.abs() + tiny)
    out["dk"] = (dk, s * ((ds_err + ds.abs() * more + sub * visible).T @ q.abs()) + final * dk.abs() + tiny)
    return out


def _sum_heads(parts, final):
    """Value and bound of a gradient that several heads add to, rounded once."""
    return sum(v for v, _ in parts), sum(b for _, b in parts)


def cross(q, k, v, lens=None, q_lens=None, scale=None, d_o=None):
    """{name: (value, bound)} of o, lse and, with d_o, dq, dk, dv; all tensors on the CPU."""
    dtype = q.dtype
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    shapes = {"o": q.shape, "lse": q.shape[:3], "dq": q.shape, "dk": k.shape, "dv": k.shape}
    names = ["o", "lse"] + (["dq", "dk", "dv"] if d_o is not None else [])
    res = {n: [torch.zeros(shapes[n], dtype=torch.float64) for _ in range(2)] for n in names}
    for b in range(B):
        L = Tk if lens is None else min(max(int(lens[b]), 0), Tk)
        n = Tq if q_lens is None else min(max(int(q_lens[b]), 0), Tq)
        for h in range(Hq):
            seen = torch.ones(n, L, dtype=torch.bool)
            r = _head(q[b, h, :n].double(), k[b, h // G, :L].double(), v[b, h // G, :L].double(), seen, scale, dtype,
                      None if d_o is None else d_o[b, h, :n].double())
            for name in names:
                head = h // G if name in ("dk", "dv") else h
                for i in range(2):
                    x = r[name][i]
                    res[name][i][b, head, :x.shape[0]] += x
    return {n: tuple(x) for n, x in res.items()}


def paged(q, k_pages, v_pages, table, lens, C=1, R=None, scale=None, new_lens=None):
    """{name: (value, bound)} of o and lse; all tensors on the CPU."""
    B, Hq, T, D = q.shape
    N, Hkv, page, _ = k_pages.shape
    G, width = Hq // Hkv, table.shape[1]
    scale = D ** -0.5 if scale is None else scale
    res = {"o": [torch.zeros(q.shape, dtype=torch.float64) for _ in range(2)],
           "lse": [torch.zeros(q.shape[:3], dtype=torch.float64) for _ in range(2)]}
    for b in range(B):
        L = min(max(int(lens[b]), 0), width * page)
        n = T if new_lens is None else min(max(int(new_lens[b]), 0), T)
        keys, values = torch.zeros(Hkv, L, D, dtype=torch.float64), torch.zeros(Hkv, L, D, dtype=torch.float64)
        there = torch.zeros(L, dtype=torch.bool)
        for j in range(L):
            e = int(table[b, j // page])
            if 0 <= e < N:
                there[j] = True
                keys[:, j], values[:, j] = k_pages[e, :, j % page].double(), v_pages[e, :, j % page].double()
        seen = torch.zeros(n, L, dtype=torch.bool)
        for i in range(n):
            at = L - n + i
            if at >= 0:
                gap = at // C - torch.arange(L) // C
                seen[i] = (gap >= 0) & there
                if R is not None:
                    seen[i] &= gap <= R
        for h in range(Hq):
            r = _head(q[b, h, :n].double(), keys[h // G], values[h // G], seen, scale, q.dtype)
            for name in res:
                for i in range(2):
                    res[name][i][b, h, :n] = r[name][i]
    return {n: tuple(x) for n, x in res.items()}


def assert_within(name, got, want_bound, finite=True):
    want, bound = want_bound
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} instead of {tuple(want.shape)}"
    assert not finite or torch.isfinite(got[torch.isfinite(want)]).all(), f"{name}: values that are not finite"
    same = got == want   # infinities among them
    off = (got - want).abs()
    bad = ~(same | (off <= bound))
    if bad.any():
        worst = torch.where(bad, off / bound.clamp(min=1e-300), 0.0)
        at = torch.unravel_index(worst.argmax(), worst.shape) if worst.dim() else ()
        at = tuple(int(i) for i in at)
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, worst at {at}: "
                             f"{float(got[at])} instead of {float(want[at])}, bound {float(bound[at])}")
