"""What comes before attention, and decoding with drafted tokens, as measurable cases: norms of queries and keys with the position
rotation (`qk_norm_rope`, forward and backward), the same on the way into a cache in pages (`paged_append_rope`), attention of a tree of
drafted tokens over the cache (`paged_tree_attention`), and keeping the accepted ones (`paged_keep`).

A case holds
  what    "rope_train" (forward + backward), "rope" (forward only), "append" (paged_append_rope), "tree", "keep"
  dtype, B, Hq, Hkv, D
  T       tokens of a sequence; for "append", "tree" and "keep" the new ones
  L       longest sequence in the cache, the new tokens counted ("append", "tree", "keep")
  lens    lengths: "full", "half" (uniform in [L/2, L]), "any" (uniform in [1, L]) or "log" (log-uniform in [min(64, L), L]); for "rope"
          and "rope_train" those of the sequences, L = T
  ragged  the new tokens of a sequence are fewer than T for some ("append", "tree")
  page    positions of a page
  rot     channels that are rotated, the first ones ("rope", "rope_train", "append")
  norm    with norms and their weights
  inter   pairs are neighbours instead of halves
  packed  q, k (and v) are views of one projection output [B, T, Hq + 2 Hkv, D]
  tree    "chain", "wide" (most tokens near the root) or "any"; shared: one tree for all sequences.  "append": the tokens are those of such a
          tree, at the positions of their depths ("" for a run of tokens)
  lse     the log-sum-exp is asked for as well ("tree")
  kept    tokens that are kept, at most ("keep")
With G = Hq / Hkv, query head h reads key head h // G.
"""
import math
import os
import sys

import torch

own = False
EPS = 1e-6


def _case(what, dtype, B, Hq, Hkv, T, D, L=0, lens="full", ragged=False, page=0, rot=0, norm=False, inter=False, packed=False, tree="",
          shared=False, lse=False, kept=0, name=None):
    c = dict(what=what, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, T=T, D=D, L=L or T, lens=lens, ragged=ragged, page=page, rot=rot, norm=norm,
             inter=inter, packed=packed, tree=tree, shared=shared, lse=lse, kept=kept)
    return c if name is None else dict(name=name, **c)


def listed():
    return [
        # a debugging-size float32 training step
        _case("rope_train", "float32", 2, 4, 4, 50, 64, lens="half", rot=64, norm=True, name="rope_train_small_fp32"),
        # a training step of long sequences with shared key heads, q and k read in place from the projection's output
        _case("rope_train", "bfloat16", 2, 32, 8, 8192, 128, rot=128, norm=True, packed=True, name="rope_train_long_bf16"),
        # a padded batch without norms, half of the channels rotated in neighbouring pairs
        _case("rope", "float16", 16, 16, 16, 1500, 64, lens="any", rot=32, inter=True, name="rope_batch_fp16"),
        # one token of one sequence: latency
        _case("append", "float16", 1, 8, 8, 1, 64, 300, page=16, rot=64, norm=True, name="append_one_token_fp16"),
        # the newest token of a serving batch, straight from the projection
        _case("append", "bfloat16", 64, 32, 8, 1, 128, 1024, "log", page=16, rot=128, packed=True, name="append_token_bf16"),
        # prompts into the cache
        _case("append", "bfloat16", 8, 32, 8, 2048, 128, 4096, "half", True, page=64, rot=128, norm=True, packed=True, name="append_prompt_bf16"),
        # a few drafted tokens of one short sequence: latency
        _case("tree", "float16", 1, 8, 8, 8, 64, 300, page=16, tree="any", shared=True, name="tree_one_sequence_fp16"),
        # a serving batch of every length, sixteen drafted tokens each, grouped heads
        _case("tree", "bfloat16", 32, 32, 8, 16, 128, 8192, "log", page=16, tree="wide", shared=True, name="tree_batch_bf16"),
        # large trees, one of its own for each sequence
        _case("tree", "bfloat16", 8, 32, 8, 64, 128, 8192, "half", True, page=64, tree="any", name="tree_large_bf16"),
        # few very long sequences
        _case("tree", "bfloat16", 2, 32, 8, 8, 128, 131072, "half", page=64, tree="any", name="tree_long_bf16"),
        # the accepted tokens of one sequence
        _case("keep", "float16", 1, 8, 8, 16, 64, 300, page=16, kept=4, name="keep_one_sequence_fp16"),
        # those of a serving batch
        _case("keep", "bfloat16", 64, 8, 8, 64, 128, 1024, "half", page=16, kept=8, name="keep_batch_bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    kv = rng.choice([h for h in (1, 2, 3, 4, 8, 12, 16) if h <= most])
    return kv * rng.choice([g for g in (1, 1, 2, 3, 4, 6, 8) if kv * g <= most]), kv


def _fits(c):
    """Whether a drawn case costs no more than the largest listed one of its kind (and its plain form's scores fit)."""
    w, cases = work(c), listed()
    if c["what"] in ("rope", "rope_train"):
        return w["bytes"] <= work(cases[1])["bytes"]
    if c["what"] in ("append", "keep"):
        cache = c["B"] * c["Hkv"] * -(-c["L"] // c["page"]) * c["page"] * c["D"]
        return cache <= 1 << 26 and w["bytes"] <= work(cases[5])["bytes"]
    slower = 16 if c["dtype"] == "float32" else 2
    scores = c["B"] * c["Hq"] * c["T"] * c["L"]
    return w["flops"] * slower <= work(cases[8])["flops"] * 2 and w["bytes"] <= 1.2e9 and scores <= 1 << 28


def draw(rng):
    while True:
        kind = rng.choice(["rope_small", "rope_long", "rope_batch", "append_token", "append_prompt", "append_tree", "tree_small", "tree_batch",
                           "tree_large", "tree_long", "keep"])
        half = rng.choice(["float16", "bfloat16"])
        any_type = rng.choice(["float32", half, half])
        lens = rng.choice(["full", "half", "any", "log"])
        ragged, packed, inter, norm, lse, shared = (rng.random() < p for p in (0.5, 0.5, 0.3, 0.6, 0.25, 0.5))
        what = rng.choice(["rope_train", "rope"])
        page = rng.choice([1, 8, 16, 16, 32, 48, 64, 100, 128, 256])
        tree = rng.choice(["chain", "wide", "any"])
        D = rng.choice([16, 32, 64, 128, 256])
        rot = rng.choice([D, D, max(16, D // 2), 16 * rng.randint(1, D // 16)])
        if kind == "rope_small":
            hq, hkv = _heads(rng, 8)
            c = _case(what, any_type, rng.randint(1, 4), hq, hkv, _log(rng, 1, 600), D, lens=lens, rot=rot, norm=norm, inter=inter, packed=packed)
        elif kind == "rope_long":
            hq, hkv = _heads(rng, 64)
            c = _case(what, half, rng.randint(1, 4), hq, hkv, _log(rng, 1000, 16384), D, lens=rng.choice(["full", lens]), rot=rot, norm=norm,
                      inter=inter, packed=packed)
        elif kind == "rope_batch":
            hq, hkv = _heads(rng, 16)
            c = _case(what, any_type, _log(rng, 4, 128), hq, hkv, _log(rng, 20, 2000), D, lens=lens, rot=rot, norm=norm, inter=inter, packed=packed)
        elif kind == "append_token":
            hq, hkv = _heads(rng, 64)
            c = _case("append", any_type, _log(rng, 1, 128), hq, hkv, rng.choice([1, 1, 1, 2, 5]), D, _log(rng, 8, 2048), lens, ragged, page, rot,
                      norm, inter, packed)
        elif kind == "append_prompt":
            hq, hkv = _heads(rng, 32)
            T = _log(rng, 16, 2048)
            c = _case("append", any_type, _log(rng, 1, 32), hq, hkv, T, D, T + _log(rng, 1, 2048), lens, ragged, page, rot, norm, inter, packed)
        elif kind == "append_tree":
            hq, hkv = _heads(rng, 32)
            T = rng.randint(2, 64)
            c = _case("append", half, _log(rng, 1, 64), hq, hkv, T, D, T + _log(rng, 1, 2048), lens, ragged, page, rot, norm, inter, packed, tree,
                      shared)
        elif kind == "tree_small":
            hq, hkv = _heads(rng, 16)
            T = _log(rng, 1, 32)
            c = _case("tree", any_type, rng.randint(1, 4), hq, hkv, T, D, T + _log(rng, 1, 1000), lens, ragged, page, tree=tree, shared=shared, lse=lse)
        elif kind == "tree_batch":
            hq, hkv = _heads(rng, 64)
            T = _log(rng, 2, 32)
            c = _case("tree", half, _log(rng, 4, 64), hq, hkv, T, rng.choice([64, 128, 256]), T + _log(rng, 128, 8192), lens, ragged, page, tree=tree,
                      shared=shared, lse=lse)
        elif kind == "tree_large":
            hq, hkv = _heads(rng, 32)
            T = _log(rng, 32, 256)
            c = _case("tree", half, _log(rng, 1, 16), hq, hkv, T, rng.choice([32, 64, 128]), T + _log(rng, 128, 8192), lens, ragged, page, tree=tree,
                      shared=shared, lse=lse)
        elif kind == "tree_long":
            hq, hkv = _heads(rng, 32)
            c = _case("tree", half, rng.randint(1, 4), hq, hkv, _log(rng, 2, 16), rng.choice([64, 128]), _log(rng, 16384, 131072), lens, False,
                      page, tree=tree, shared=shared, lse=lse)
        else:
            hkv = rng.choice([1, 2, 4, 8, 16])
            T = _log(rng, 2, 128)
            c = _case("keep", any_type, _log(rng, 1, 128), hkv, hkv, T, D, T + _log(rng, 1, 2048), lens, page=page, kept=rng.randint(1, (T + 1) // 2))
        if _fits(c):
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _lengths(B, longest, how, gen):
    u = torch.rand(B, generator=gen, dtype=torch.float64)
    if how == "full":
        n = torch.full((B,), longest)
    elif how == "log":
        lo = min(64, longest)
        n = torch.floor(lo * torch.exp(u * math.log(longest / lo)))
    else:
        lo = longest // 2 if how == "half" else 1
        n = lo + torch.floor(u * (longest - lo + 1))
    n = n.to(torch.int32).clamp(1, longest)
    if how != "full":
        n[int(torch.randint(B, (1,), generator=gen))] = longest   # a padded batch is as long as its longest sequence
    return n


def _tables(positions, rot, dev):
    """cos and sin of every position's angles, [positions, rot / 2]."""
    rate = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _trees(n, T, how, gen):
    """[n, T, T]: which tokens each one sees: itself and its ancestors, which lie before it."""
    seen = torch.zeros(n, T, T, dtype=torch.bool)
    each = torch.arange(n)
    for i in range(T):
        if how == "chain":
            parent = torch.full((n,), i - 1)
        else:   # a token before it (or the context, -1); "wide" prefers early ones
            u = torch.rand(n, generator=gen, dtype=torch.float64)
            parent = torch.floor((u * u if how == "wide" else u) * (i + 1)).long() - 1
        seen[:, i] = torch.where((parent >= 0)[:, None], seen[each, parent.clamp(min=0)], False)
        seen[:, i, i] = True
    return seen


def prepare(case, seed):
    c = case
    dev, dt = torch.device("cuda"), getattr(torch, c["dtype"])
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev).to(dt)

    B, Hq, Hkv, T, D, L, page = (c[n] for n in ("B", "Hq", "Hkv", "T", "D", "L", "page"))
    s = dict(c=c)
    if c["what"] in ("rope", "rope_train", "append"):
        if c["packed"]:
            qkv = randn(B, T, Hq + 2 * Hkv, D).transpose(1, 2)
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        else:
            s["q"], s["k"], s["v"] = randn(B, Hq, T, D), randn(B, Hkv, T, D), randn(B, Hkv, T, D)
        s["cos"], s["sin"] = _tables(L, c["rot"], dev)
        s["wq"] = s["wk"] = None
        if c["norm"]:
            s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(dt) for _ in range(2))
    if not page:
        del s["v"]
        s["lens"] = None if c["lens"] == "full" else _lengths(B, T, c["lens"], host).to(dev)
        if c["what"] == "rope_train":
            s["g_q"], s["g_k"] = randn(B, Hq, T, D), randn(B, Hkv, T, D)
            for n in ("q", "k", "wq", "wk"):
                if s[n] is not None:
                    s[n] = s[n].detach().requires_grad_()
        return s
    lens = _lengths(B, L, c["lens"], host)
    new = None
    if c["ragged"]:
        new = torch.randint(1, T + 1, (B,), generator=host, dtype=torch.int32)
        new[int(torch.randint(B, (1,), generator=host))] = T
    count = torch.full_like(lens, T) if new is None else new
    lens = torch.maximum(lens, count)   # lengths count the new tokens
    pages = (lens + page - 1) // page
    width = -(-L // page)
    total = (int(pages.sum()) if c["what"] == "tree" else B * width) + 7   # (elsewhere the whole cache is an output)
    order = torch.randperm(total, generator=host).to(torch.int32)   # pages of a cache that has been in use for a while
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages.tolist()):
        table[b, :n] = order[at:at + n]
        at += n
    s["lens"], s["new"], s["table"] = lens.to(dev), None if new is None else new.to(dev), table.to(dev)
    s["k_pages"], s["v_pages"] = randn(total, Hkv, page, D), randn(total, Hkv, page, D)
    if c["tree"]:
        seen = _trees(1 if c["shared"] else B, T, c["tree"], host)
        s["tree"] = (seen[0] if c["shared"] else seen).to(dev)
    if c["what"] == "tree":
        s["q"] = randn(B, Hq, T, D)
    elif c["what"] == "append":
        s["positions"] = None
        if c["tree"]:
            depth = seen.sum(-1) - 1
            s["positions"] = ((lens - count)[:, None] + depth).to(torch.int32).to(dev)
    else:   # paths down trees; no place that is written is another token's (a pass can be made again)
        s["first"] = (lens - T).to(dev)
        m = c["kept"]
        kept = torch.full((B, m), -1, dtype=torch.int32)
        for b in range(B):
            n = int(torch.randint(1, m + 1, (1,), generator=host))
            kept[b, :n] = n + torch.randperm(T - n, generator=host)[:n].sort().values if T >= 2 * n else torch.arange(n)
        s["kept"] = kept.to(dev)
    return s


# ---- the calls ----------------------------------------------------------------------------------------------------

_entries = None


def _own():
    global _entries
    if _entries is None:
        import kernels_amd

        path = os.path.dirname(os.path.abspath(kernels_amd.__file__))
        if path not in sys.path:
            sys.path.insert(0, path)
        from paged_attention import paged_append_rope, paged_keep, paged_tree_attention
        from qk_norm_rope import qk_norm_rope

        _entries = qk_norm_rope, paged_append_rope, paged_tree_attention, paged_keep
    return _entries


def run(state):
    c = state["c"]
    return (_run_own if own else _run_plain)(c, state)


def _run_own(c, s):
    qk_norm_rope, paged_append_rope, paged_tree_attention, paged_keep = _own()
    eps = EPS if c["norm"] else None
    if c["what"] == "append":
        q = paged_append_rope(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cos"], s["sin"], s["wq"], s["wk"],
                              new_lens=s["new"], positions=s["positions"], eps=eps, interleaved=c["inter"])
        return q, s["k_pages"], s["v_pages"]
    if c["what"] == "tree":
        return paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["tree"], new_lens=s["new"], return_lse=c["lse"])
    if c["what"] == "keep":
        paged_keep(s["k_pages"], s["v_pages"], s["table"], s["first"], s["kept"])
        return s["k_pages"], s["v_pages"]
    q, k = qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["wq"], s["wk"], lens=s["lens"], eps=eps, interleaved=c["inter"])
    if c["what"] == "rope":
        return q, k
    leaves = [s[n] for n in ("q", "k", "wq", "wk") if s[n] is not None]
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["g_q"], s["g_k"])))


# ---- the plain forms: 32 bits, whatever the inputs' type ------------------------------------------------------------

def _turn(x, cos, sin, rot, inter):
    """x [..., D] with the pairs of its first `rot` channels turned by the angles of cos and sin [..., rot / 2]."""
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rot:]), -1) if rot < x.shape[-1] else y


def _unit(x, norm):
    """x over its root mean square, and the factor."""
    if not norm:
        return x, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _run_plain(c, s):
    if c["what"] == "append":
        return _append_plain(c, s)
    if c["what"] == "tree":
        return _tree_plain(c, s)
    if c["what"] == "keep":
        return _keep_plain(c, s)
    rot, inter = c["rot"], c["inter"]
    T = c["T"]
    live = None if s["lens"] is None else (torch.arange(T, device=s["q"].device) < s["lens"][:, None])[:, None, :, None]
    cos, sin = s["cos"][:T], s["sin"][:T]
    out, grads, weights = [], [], []
    with torch.no_grad():
        for n in ("q", "k"):
            x, w = s[n].float(), s["w" + n]
            unit, r = _unit(x, c["norm"])
            y = _turn(unit if w is None else unit * w.float(), cos, sin, rot, inter)
            out.append((y if live is None else torch.where(live, y, 0.0)).to(s[n].dtype))
            if c["what"] == "rope":
                continue
            g = s["g_" + n].float()
            g = _turn(g if live is None else torch.where(live, g, 0.0), cos, -sin, rot, inter)
            if c["norm"]:
                weights.append((g * unit).sum((0, 1, 2)).to(w.dtype))
                h = g * w.float()
                g = r * (h - unit * (h * unit).mean(-1, keepdim=True))
            grads.append(g.to(s[n].dtype))
    return (*out, *grads, *weights)


def _new_tokens(c, s):
    """(b, t, position) of the new tokens that there are."""
    lens = s["lens"][:, None].long()
    count = s["new"][:, None] if s["new"] is not None else c["T"]
    i = torch.arange(c["T"], device=lens.device)
    b, t = torch.nonzero((i < count).expand(len(lens), c["T"]), as_tuple=True)
    return b, t, (lens - count + i).expand(len(lens), c["T"])[b, t]


def _append_plain(c, s):
    page = c["page"]
    b, t, at = _new_tokens(c, s)
    where = at if s["positions"] is None else s["positions"].expand(c["B"], c["T"])[b, t].long()
    cos, sin = s["cos"][where][:, None], s["sin"][where][:, None]
    turned = []
    for n in ("q", "k"):
        x = _unit(s[n][b, :, t].float(), c["norm"])[0]
        x = x if s["w" + n] is None else x * s["w" + n].float()
        turned.append(_turn(x, cos, sin, c["rot"], c["inter"]).to(s[n].dtype))
    q = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    q[b, :, t] = turned[0]
    to = s["table"][b, at // page].long()
    s["k_pages"][to, :, at % page] = turned[1]
    s["v_pages"][to, :, at % page] = s["v"][b, :, t]
    return q, s["k_pages"], s["v_pages"]


def _tree_plain(c, s):
    B, Hq, Hkv, T, D, page = (c[n] for n in ("B", "Hq", "Hkv", "T", "D", "page"))
    G, dev, lens = Hq // Hkv, s["q"].device, s["lens"][:, None].long()
    width = s["table"].shape[1]
    span = width * page
    pages = s["table"].clamp(min=0).long()
    at = torch.arange(span, device=dev)
    k, v = (x[pages].transpose(1, 2).reshape(B, Hkv, span, D).float() for x in (s["k_pages"], s["v_pages"]))
    v = torch.where((at < lens)[:, None, :, None], v, 0.0)
    count = s["new"][:, None].long() if s["new"] is not None else torch.full_like(lens, T)
    live = torch.arange(T, device=dev) < count
    first = lens - count
    new = at - first                                                     # [B, span]: the drafted token that a position holds
    tree = s["tree"].expand(B, T, T)
    seen = torch.gather(tree, 2, new.clamp(0, T - 1)[:, None].expand(B, T, span)) & (new >= 0)[:, None] & (new < count)[:, None]
    seen |= (new < 0)[:, None]
    q = s["q"].float().reshape(B, Hkv, G * T, D)
    x = (torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5).reshape(B, Hkv, G, T, span)
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, G * T, span), v).reshape(B, Hkv, G, T, D) / total
    o = torch.where(live[:, None, :, None], o.reshape(B, Hq, T, D), 0.0).to(s["q"].dtype)
    if not c["lse"]:
        return o
    lse = (top + torch.log(total)).reshape(B, Hq, T) * math.log2(math.e)
    return o, torch.where(live[:, None], lse, 0.0)


def _keep_plain(c, s):
    page, kept = c["page"], s["kept"].long()
    b, i = torch.nonzero(kept >= 0, as_tuple=True)
    first = s["first"].long()[b]
    src, dst = first + kept[b, i], first + i
    from_page, to_page = s["table"][b, src // page].long(), s["table"][b, dst // page].long()
    for x in (s["k_pages"], s["v_pages"]):
        x[to_page, :, dst % page] = x[from_page, :, src % page]
    return s["k_pages"], s["v_pages"]


# ---- work and exact results ---------------------------------------------------------------------------------------

def _share(c):
    """The mean length over the longest: lengths are drawn with the inputs."""
    share = {"full": 1.0, "half": 0.75, "any": 0.5, "log": 0.5}[c["lens"]]
    if c["lens"] == "log" and c["L"] > 64:
        share = (1 - 64 / c["L"]) / math.log(c["L"] / 64)
    return share + (1 - share) / c["B"]   # one sequence has the whole length


def work(case):
    c = case
    es = 4 if c["dtype"] == "float32" else 2
    new = c["T"] * (0.5 + 0.5 / c["T"] if c["ragged"] else 1.0)
    row = c["B"] * c["D"] * es
    if c["what"] in ("rope", "rope_train"):
        live = c["T"] * _share(c)   # rows of padding are written, not read
        train = c["what"] == "rope_train"
        heads = c["Hq"] + c["Hkv"]
        each = (2 * live + 2 * c["T"]) if train else (live + c["T"])
        return {"bytes": int(row * heads * each + 4 * c["T"] * c["rot"]),
                "flops": int(c["B"] * heads * live * (3 * c["rot"] + (4 * c["D"] if c["norm"] else 0)) * (3 if train else 1))}
    if c["what"] == "append":
        rows = c["Hq"] + c["Hkv"]
        return {"bytes": int(row * ((c["Hq"] + 4 * c["Hkv"]) * new + c["Hq"] * c["T"])),
                "flops": int(c["B"] * rows * new * (3 * c["rot"] + (4 * c["D"] if c["norm"] else 0)))}
    if c["what"] == "keep":
        return {"bytes": int(4 * row * c["Hkv"] * (c["kept"] + 1) / 2), "flops": 0}
    keys = max(c["L"] * _share(c), new)
    return {"bytes": int(row * (2 * c["Hkv"] * keys + c["Hq"] * (new + c["T"])) + c["T"] * c["T"] * (1 if c["shared"] else c["B"])),
            "flops": int(4 * c["B"] * c["Hq"] * new * keys * c["D"])}


def _turned_exactly(x, w, cos, sin, c):
    """[..., D] in 64 bits: the pairs as complex numbers."""
    rot = c["rot"]
    if c["norm"]:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["D"] + EPS) * w
    if c["inter"]:
        pair = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * torch.complex(cos, sin)
        y = torch.view_as_real(pair).flatten(-2)
    else:
        pair = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * torch.complex(cos, sin)
        y = torch.cat((pair.real, pair.imag), -1)
    return torch.cat((y, x[..., rot:]), -1)


def exact(case, seed):
    """The definition in 64 bits, one sequence at a time; gradients by differentiating it."""
    c, s = case, prepare(case, seed)
    B, Hq, Hkv, T, D, page = (c[n] for n in ("B", "Hq", "Hkv", "T", "D", "page"))
    dev = (s["q"] if "q" in s else s["k_pages"]).device
    lens = [T] * B if s["lens"] is None else s["lens"].tolist()
    if c["what"] in ("rope", "rope_train"):
        train = c["what"] == "rope_train"
        out, grads, weights = [], [], []
        for n in ("q", "k"):
            y, dx, dw = (torch.zeros(s[n].shape if d else D, dtype=torch.float64, device=dev) for d in (1, 1, 0))
            for b in range(B):
                live = lens[b]
                x = s[n][b, :, :live].detach().double().requires_grad_(train)
                w = s["w" + n].detach().double().requires_grad_(train) if c["norm"] else None
                o = _turned_exactly(x, w, s["cos"][:live].double(), s["sin"][:live].double(), c)
                y[b, :, :live] = o.detach()
                if train:
                    got = torch.autograd.grad(o, [x] + ([w] if c["norm"] else []), s["g_" + n][b, :, :live].double())
                    dx[b, :, :live] = got[0]
                    if c["norm"]:
                        dw += got[1]
            out.append(y), grads.append(dx), weights.append(dw)
        return (*out, *grads, *(weights if c["norm"] else [])) if train else tuple(out)
    new = [T] * B if s["new"] is None else s["new"].tolist()
    table = s["table"].tolist()
    if c["what"] == "append":
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"]
        for b in range(B):
            n, first = new[b], lens[b] - new[b]
            at = torch.arange(first, first + n, device=dev) if s["positions"] is None else s["positions"][b if len(s["positions"]) > 1 else 0, :n].long()
            cos, sin = s["cos"][at].double(), s["sin"][at].double()
            w = (s["wq"].double(), s["wk"].double()) if c["norm"] else (None, None)
            q[b, :, :n] = _turned_exactly(s["q"][b, :, :n].double(), w[0], cos, sin, c)
            k = _turned_exactly(s["k"][b, :, :n].double(), w[1], cos, sin, c)
            t = 0
            while t < n:   # page by page
                slot = (first + t) % page
                m = min(page - slot, n - t)
                to = table[b][(first + t) // page]
                k_pages[to, :, slot:slot + m] = k[:, t:t + m]
                v_pages[to, :, slot:slot + m] = s["v"][b, :, t:t + m]
                t += m
        return q, k_pages, v_pages
    if c["what"] == "keep":
        kept, first = s["kept"].tolist(), s["first"].tolist()
        for b in range(B):
            for i, j in enumerate(kept[b]):
                if j >= 0:
                    src, dst = first[b] + j, first[b] + i
                    for x in (s["k_pages"], s["v_pages"]):
                        x[table[b][dst // page], :, dst % page] = x[table[b][src // page], :, src % page]
        return s["k_pages"], s["v_pages"]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=dev)
    lse = torch.zeros(B, Hq, T, dtype=torch.float64, device=dev)
    for b in range(B):
        n, L = new[b], lens[b]
        to = s["table"][b, :-(-L // page)].long()
        keys, values = (x[to].transpose(0, 1).flatten(1, 2)[:, :L] for x in (s["k_pages"], s["v_pages"]))
        hidden = torch.zeros(n, L, dtype=torch.bool, device=dev)
        hidden[:, L - n:] = ~(s["tree"] if c["shared"] else s["tree"][b])[:n, :n]
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            x = (s["q"][b, heads, :n].double() @ keys[h].double().T) / math.sqrt(D)
            x = x.masked_fill(hidden, -math.inf)
            out[b, heads, :n] = torch.softmax(x, -1) @ values[h].double()
            lse[b, heads, :n] = torch.logsumexp(x, -1) / math.log(2)
    return (out, lse) if c["lse"] else out
