"""Attention over keys that are not the queries' own, as measurable cases: an encoder's states
(`cross_attention`, forward and backward) and a cache in pages (`paged_attention` for the newest
tokens of every sequence, `paged_append`, which puts their keys and values there).

A case holds
  what    "cross_train" (forward + backward), "cross" (forward only), "paged", "append"
  dtype, B, Hq, Hkv, D
  Tq      queries of a batch entry; for "paged" and "append" the new tokens of a sequence
  Tk      keys of a batch entry; for "paged" and "append" the longest sequence
  lens    lengths of the key sequences: "full", "half" (uniform in [Tk/2, Tk]), "any" (uniform in
          [1, Tk]) or "log" (log-uniform in [min(64, Tk), Tk])
  ragged  the queries (new tokens) of a batch entry are fewer than Tq for some
  lse     the log-sum-exp is asked for as well ("cross" and "paged")
  packed  k and v are views of one [B, Tk, 2, Hkv, D] projection output ("cross" ones)
  page    positions of a page ("paged", "append")
  C, R    chunk length and number of earlier chunks a new token sees ("paged"; C = 1 with R < 0: all
          positions up to its own)
With G = Hq / Hkv, query head h reads key head h // G.
"""
import math
import os
import sys

import torch

own = False


def _case(what, dtype, B, Hq, Hkv, Tq, Tk, D, lens="full", ragged=False, lse=False, packed=False, page=0, C=0, R=0, name=None):
    c = dict(what=what, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Tq=Tq, Tk=Tk, D=D, lens=lens, ragged=ragged, lse=lse, packed=packed,
             page=page, C=C, R=R)
    return c if name is None else dict(name=name, **c)


def listed():
    return [
        # a debugging-size float32 training step
        _case("cross_train", "float32", 2, 4, 4, 50, 512, 64, "half", True, name="cross_train_small_fp32"),
        # text decoder over the states of a speech encoder, batch of utterances, both sides padded
        _case("cross_train", "float16", 32, 12, 12, 224, 1500, 64, "half", True, name="cross_train_speech_fp16"),
        # long queries over long states with shared key heads
        _case("cross_train", "bfloat16", 2, 32, 8, 4096, 8192, 128, name="cross_train_long_bf16"),
        # wide heads, k and v read in place from the projection's output
        _case("cross_train", "bfloat16", 4, 8, 8, 500, 2048, 256, "any", packed=True, name="cross_train_wide_bf16"),
        # many queries over a short conditioning sequence
        _case("cross", "float16", 8, 16, 16, 4096, 77, 64, "any", name="cross_short_states_fp16"),
        # one decoding step: a single query per sequence over its encoder's states
        _case("cross", "float16", 16, 12, 12, 1, 1500, 64, "half", name="cross_one_token_fp16"),
        # one decoding step of one short sequence: latency
        _case("paged", "float16", 1, 8, 8, 1, 300, 64, page=16, C=1, R=-1, name="paged_one_sequence_fp16"),
        # a serving batch of every length, grouped heads
        _case("paged", "bfloat16", 64, 32, 8, 1, 8192, 128, "log", page=16, C=1, R=-1, name="paged_batch_bf16"),
        # few very long sequences
        _case("paged", "bfloat16", 2, 32, 8, 1, 131072, 128, "half", page=64, C=1, R=-1, name="paged_long_bf16"),
        # streaming inference: a chunk of frames arrives and sees the chunks before it
        _case("paged", "float16", 32, 8, 8, 32, 3000, 64, "any", page=32, C=32, R=9, name="paged_chunk_fp16"),
        # the newest token of a serving batch into the cache
        _case("append", "bfloat16", 64, 8, 8, 1, 1024, 128, "log", page=16, name="append_token_bf16"),
        # prompts into the cache
        _case("append", "bfloat16", 8, 8, 8, 2048, 4096, 128, "half", True, page=64, name="append_prompt_bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    kv = rng.choice([h for h in (1, 2, 3, 4, 8, 12, 16) if h <= most])
    return kv * rng.choice([g for g in (1, 1, 1, 2, 3, 4, 6, 8, 16) if kv * g <= most]), kv


def _fits(c):
    """Whether a drawn case costs no more than the largest listed one."""
    w, most = work(c), work(listed()[2])
    slower = 16 if c["dtype"] == "float32" else 2 if c["D"] < 128 else 1
    scores = c["B"] * c["Hq"] * c["Tq"] * c["Tk"]
    if c["what"] == "append":
        return c["B"] * c["Hkv"] * c["Tk"] * c["D"] <= 1 << 27
    return w["flops"] * slower <= most["flops"] and w["bytes"] <= 2e9 and (c["what"] != "paged" or scores <= 1 << 29)


def draw(rng):
    while True:
        kind = rng.choice(["cross_small", "cross_text", "cross_long", "cross_short", "cross_one", "paged_small", "paged_batch",
                           "paged_long", "paged_chunk", "append"])
        half = rng.choice(["float16", "bfloat16"])
        lens = rng.choice(["full", "half", "any", "log"])
        ragged, lse, packed = rng.random() < 0.5, rng.random() < 0.25, rng.random() < 0.25
        what = rng.choice(["cross_train", "cross"])
        page = rng.choice([1, 8, 16, 16, 32, 48, 64, 100, 128, 256])
        if what == "cross_train":
            lse = False
        if kind == "cross_small":     # a few short sequences of any type
            hq, hkv = _heads(rng, 8)
            c = _case(what, rng.choice(["float32", half]), rng.randint(1, 4), hq, hkv, _log(rng, 1, 300), _log(rng, 1, 600),
                      rng.choice([16, 32, 64, 128, 256]), lens, ragged, lse, packed)
        elif kind == "cross_text":    # a text's queries over the states of speech or images
            hq, hkv = _heads(rng, 16)
            c = _case(what, half, _log(rng, 4, 64), hq, hkv, _log(rng, 20, 448), _log(rng, 200, 3000), rng.choice([32, 64, 128]),
                      lens, ragged, lse, packed)
        elif kind == "cross_long":    # long on both sides
            hq, hkv = _heads(rng, 32)
            c = _case(what, half, rng.randint(1, 4), hq, hkv, _log(rng, 512, 8192), _log(rng, 1024, 16384), rng.choice([64, 128, 256]),
                      lens, ragged, lse, packed)
        elif kind == "cross_short":   # many queries, few keys
            hq, hkv = _heads(rng, 16)
            c = _case(what, half, rng.randint(1, 16), hq, hkv, _log(rng, 1000, 9000), _log(rng, 4, 256), rng.choice([32, 64, 128]),
                      lens, ragged, lse, packed)
        elif kind == "cross_one":     # the decoding step of a decoder over its encoder
            hq, hkv = _heads(rng, 32)
            c = _case("cross", rng.choice([half, half, "float32"]), _log(rng, 1, 64), hq, hkv, rng.choice([1, 1, 1, 2, 4]),
                      _log(rng, 50, 20000), rng.choice([32, 64, 128]), lens, False, lse, packed)
        elif kind == "paged_small":
            hq, hkv = _heads(rng, 16)
            c = _case("paged", rng.choice([half, "float32"]), rng.randint(1, 4), hq, hkv, 1, _log(rng, 1, 1000),
                      rng.choice([16, 32, 64, 128, 256]), lens, False, lse, page=page, C=1, R=-1)
        elif kind == "paged_batch":
            hq, hkv = _heads(rng, 64)
            c = _case("paged", half, _log(rng, 4, 128), hq, hkv, rng.choice([1, 1, 1, 2, 5]), _log(rng, 128, 8192),
                      rng.choice([64, 128, 256]), lens, ragged, lse, page=page, C=1, R=rng.choice([-1, -1, _log(rng, 64, 4096)]))
        elif kind == "paged_long":
            hq, hkv = _heads(rng, 32)
            c = _case("paged", half, rng.randint(1, 4), hq, hkv, 1, _log(rng, 16384, 131072), rng.choice([64, 128]), lens, False, lse,
                      page=page, C=1, R=-1)
        elif kind == "paged_chunk":   # chunks of a stream
            hq, hkv = _heads(rng, 16)
            C = _log(rng, 4, 64)
            c = _case("paged", half, _log(rng, 1, 64), hq, hkv, C, _log(rng, C, 4000), rng.choice([32, 64, 128]), lens, False, lse,
                      page=page, C=C, R=rng.randint(0, 9))
        else:
            hkv = rng.choice([1, 2, 4, 8, 16])
            tq = rng.choice([1, 1, 2, _log(rng, 16, 2048)])
            c = _case("append", rng.choice([half, "float32"]), _log(rng, 1, 128), hkv, hkv, tq, tq + _log(rng, 1, 2048),
                      rng.choice([32, 64, 128]), lens, ragged, page=page)
        if _fits(c):
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _lengths(c, gen):
    B, T, how = c["B"], c["Tk"], c["lens"]
    u = torch.rand(B, generator=gen, dtype=torch.float64)
    if how == "full":
        n = torch.full((B,), T)
    elif how == "log":
        lo = min(64, T)
        n = torch.floor(lo * torch.exp(u * math.log(T / lo)))
    else:
        lo = T // 2 if how == "half" else 1
        n = lo + torch.floor(u * (T - lo + 1))
    n = n.to(torch.int32).clamp(1, T)
    if how != "full":
        n[int(torch.randint(B, (1,), generator=gen))] = T   # a padded batch is as long as its longest sequence
    return n


def prepare(case, seed):
    c = case
    dev, dt = torch.device("cuda"), getattr(torch, c["dtype"])
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev).to(dt)

    B, Hq, Hkv, Tq, Tk, D = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    lens = _lengths(c, host)
    q_lens = None
    if c["ragged"]:
        q_lens = torch.randint(1, Tq + 1, (B,), generator=host, dtype=torch.int32)
        q_lens[int(torch.randint(B, (1,), generator=host))] = Tq
    s = dict(c=c, lens=lens.to(dev) if c["lens"] != "full" or c["page"] else None,
             q_lens=None if q_lens is None else q_lens.to(dev))
    if not c["page"]:
        s["q"] = randn(B, Hq, Tq, D)
        if c["packed"]:
            kv = randn(B, Tk, 2, Hkv, D)
            s["k"], s["v"] = (kv[:, :, i].transpose(1, 2) for i in range(2))
        else:
            s["k"], s["v"] = randn(B, Hkv, Tk, D), randn(B, Hkv, Tk, D)
        if c["what"] == "cross_train":
            s["d_o"] = randn(B, Hq, Tq, D)
            s["q"].requires_grad_(), s["k"].requires_grad_(), s["v"].requires_grad_()
        return s
    # lengths count the new tokens, of which a sequence has q_lens (or Tq)
    lens = torch.maximum(lens, torch.full_like(lens, Tq) if q_lens is None else q_lens)
    s["lens"] = lens.to(dev)
    page = c["page"]
    pages = (lens + page - 1) // page
    width = -(-max(Tk, Tq) // page)
    total = B * width if c["what"] == "append" else int(pages.sum())   # (the whole cache is an output of "append")
    order = torch.randperm(total + 7, generator=host).to(torch.int32)   # pages of a cache that has been in use for a while
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages.tolist()):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table.to(dev)
    s["k_pages"], s["v_pages"] = randn(total + 7, Hkv, page, D), randn(total + 7, Hkv, page, D)
    if c["what"] == "append":
        s["k"], s["v"] = randn(B, Hkv, Tq, D), randn(B, Hkv, Tq, D)
    else:
        s["q"] = randn(B, Hq, Tq, D)
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
        from cross_attention import cross_attention
        from paged_attention import paged_append, paged_attention

        _entries = cross_attention, paged_attention, paged_append
    return _entries


def run(state):
    c = state["c"]
    return (_run_own if own else _run_plain)(c, state)


def _run_own(c, s):
    cross_attention, paged_attention, paged_append = _own()
    if c["what"] == "append":
        paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], new_lens=s["q_lens"])
        return s["k_pages"], s["v_pages"]
    if c["what"] == "paged":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], c["C"], None if c["R"] < 0 else c["R"],
                               new_lens=s["q_lens"], return_lse=c["lse"])
    out = cross_attention(s["q"], s["k"], s["v"], s["lens"], q_lens=s["q_lens"], return_lse=c["lse"])
    if c["what"] == "cross":
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_o"]))


# ---- the plain forms: 32 bits, whatever the inputs' type ------------------------------------------------------------

def _softmax(scores, seen):
    """Probabilities over the keys that are seen, zeros in a row that sees none, and the base-2 log-sum-exp."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1) * math.log2(math.e)
    return p / torch.where(total == 0, 1.0, total), lse


def _run_plain(c, s):
    if c["what"] == "append":
        return _append_plain(c, s)
    if c["what"] == "paged":
        return _paged_plain(c, s)
    B, Hq, Hkv, Tq, Tk, D = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    G, scale, dt = Hq // Hkv, D ** -0.5, s["q"].dtype
    step = max(1, (1 << 28) // (Hq * Tq * Tk))   # batch entries whose scores fit in a GiB
    train = c["what"] == "cross_train"
    parts = []
    with torch.no_grad():
        for b in range(0, B, step):
            e = min(B, b + step)
            q = s["q"][b:e].float().reshape(e - b, Hkv, G * Tq, D)
            k, v = s["k"][b:e].float(), s["v"][b:e].float()
            at_k, at_q = torch.arange(Tk, device=q.device), torch.arange(Tq, device=q.device).repeat(G)
            seen = (at_k < s["lens"][b:e, None] if s["lens"] is not None else (at_k >= 0).expand(e - b, Tk))[:, None, None, :]
            live = (at_q < s["q_lens"][b:e, None] if s["q_lens"] is not None else (at_q >= 0).expand(e - b, G * Tq))[:, None, :, None]
            p, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen)
            o = torch.where(live, torch.matmul(p, v), 0.0)
            part = [o.reshape(e - b, Hq, Tq, D).to(dt)]
            if c["lse"]:
                part.append(torch.where(live.squeeze(-1), lse, 0.0).reshape(e - b, Hq, Tq))
            if train:
                g = torch.where(live, s["d_o"][b:e].float().reshape(e - b, Hkv, G * Tq, D), 0.0)
                dv = torch.matmul(p.transpose(-1, -2), g)
                ds = torch.matmul(g, v.transpose(-1, -2))
                ds = p.mul_(ds.sub_((o * g).sum(-1, keepdim=True))).mul_(scale)
                dq = torch.where(live, torch.matmul(ds, k), 0.0)
                dk = torch.matmul(ds.transpose(-1, -2), q)
                part += [dq.reshape(e - b, Hq, Tq, D).to(dt), dk.to(dt), dv.to(dt)]
            parts.append(part)
    out = [torch.cat(x) if len(parts) > 1 else x[0] for x in zip(*parts)]
    return out[0] if len(out) == 1 else tuple(out)


def _paged_plain(c, s):
    B, Hq, Hkv, Tn, D, page = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "D", "page"))
    G, C, R = Hq // Hkv, c["C"], c["R"]
    dev, lens = s["q"].device, s["lens"][:, None]
    width = s["table"].shape[1]
    pages = s["table"].clamp(min=0).long()
    at = torch.arange(width * page, device=dev)
    # [B, width, Hkv, page, D] -> [B, Hkv, width * page, D]
    k, v = (x[pages].transpose(1, 2).reshape(B, Hkv, width * page, D).float() for x in (s["k_pages"], s["v_pages"]))
    v = torch.where((at < lens)[:, None, :, None], v, 0.0)
    count = s["q_lens"][:, None] if s["q_lens"] is not None else torch.full_like(lens, Tn)
    i = torch.arange(Tn, device=dev)
    live = i < count
    chunk = torch.div(lens - count + i, C, rounding_mode="floor")
    gap = chunk[:, :, None] - torch.div(at, C, rounding_mode="floor")
    seen = (gap >= 0) & (at < lens)[:, None]
    if R >= 0:
        seen &= gap <= R
    q = s["q"].float().reshape(B, Hkv, G, Tn, D)
    p, lse = _softmax(torch.matmul(q.reshape(B, Hkv, G * Tn, D), k.transpose(-1, -2)).reshape(B, Hkv, G, Tn, -1) * D ** -0.5,
                      seen[:, None, None])
    o = torch.matmul(p.reshape(B, Hkv, G * Tn, -1), v).reshape(B, Hq, Tn, D)
    o = torch.where(live[:, None, :, None], o, 0.0).to(s["q"].dtype)
    if not c["lse"]:
        return o
    return o, torch.where(live[:, None], lse.reshape(B, Hq, Tn), 0.0)


def _append_plain(c, s):
    Tn, page = c["Tq"], c["page"]
    lens = s["lens"][:, None].long()
    count = s["q_lens"][:, None] if s["q_lens"] is not None else Tn
    i = torch.arange(Tn, device=lens.device)
    b, t = torch.nonzero((i < count).expand(len(lens), Tn), as_tuple=True)
    at = (lens - count + i).expand(len(lens), Tn)[b, t]
    to = s["table"][b, at // page].long()
    s["k_pages"][to, :, at % page] = s["k"][b, :, t]
    s["v_pages"][to, :, at % page] = s["v"][b, :, t]
    return s["k_pages"], s["v_pages"]


# ---- work and exact results ---------------------------------------------------------------------------------------

def work(case):
    c = case
    es = 4 if c["dtype"] == "float32" else 2
    # lengths are drawn with the inputs: counted as their mean
    share = {"full": 1.0, "half": 0.75, "any": 0.5, "log": 0.5}[c["lens"]]
    if c["lens"] == "log" and c["Tk"] > 64:
        share = (1 - 64 / c["Tk"]) / math.log(c["Tk"] / 64)
    share += (1 - share) / c["B"]   # one sequence has the whole length
    new = c["Tq"] * (0.5 + 0.5 / c["Tq"] if c["ragged"] else 1.0)
    row = c["B"] * c["D"] * es
    if c["what"] == "append":
        return {"bytes": int(4 * row * c["Hkv"] * new), "flops": 0}
    if c["what"] == "paged":
        keys = max(c["Tk"] * share, new)
        if c["R"] >= 0:
            keys = min(keys, c["C"] * (c["R"] + 1) + (new if c["C"] == 1 else 0))
        return {"bytes": int(2 * row * (c["Hkv"] * keys + c["Hq"] * new)),
                "flops": int(4 * c["B"] * c["Hq"] * new * keys * c["D"])}
    keys = c["Tk"] * share
    train = c["what"] == "cross_train"
    tensors_q, tensors_k = (4, 4) if train else (2, 2)   # q, o, d_o, dq and k, v, dk, dv
    return {"bytes": int(row * (tensors_q * c["Hq"] * new + tensors_k * c["Hkv"] * keys)),
            "flops": int((14 if train else 4) * c["B"] * c["Hq"] * new * keys * c["D"])}


def exact(case, seed):
    """The definition in 64 bits, one sequence and key head at a time; gradients by differentiating it."""
    c, s = case, prepare(case, seed)
    B, Hq, Hkv, Tq, Tk, D = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    G = Hq // Hkv
    n_q = s["q_lens"].tolist() if s["q_lens"] is not None else [Tq] * B
    n_k = s["lens"].tolist() if s["lens"] is not None else [Tk] * B
    if c["what"] == "append":
        table, page = s["table"].tolist(), c["page"]
        for b in range(B):
            first = n_k[b] - n_q[b]
            t = 0
            while t < n_q[b]:   # page by page
                slot = (first + t) % page
                n = min(page - slot, n_q[b] - t)
                to = table[b][(first + t) // page]
                for cache, x in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
                    cache[to, :, slot:slot + n] = x[b, :, t:t + n]
                t += n
        return s["k_pages"], s["v_pages"]
    out = torch.zeros(B, Hq, Tq, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(B, Hq, Tq, dtype=torch.float64, device=s["q"].device)
    train = c["what"] == "cross_train"
    if train:
        grads = [torch.zeros(s[n].shape, dtype=torch.float64, device=s["q"].device) for n in ("q", "k", "v")]
    for b in range(B):
        nq, nk = n_q[b], n_k[b]
        if c["page"]:
            to = s["table"][b, :-(-nk // c["page"])].long()
            keys, values = (x[to].transpose(0, 1).flatten(1, 2)[:, :nk] for x in (s["k_pages"], s["v_pages"]))
            pos_q = torch.arange(nk - nq, nk, device=out.device) // c["C"]
            pos_k = torch.arange(nk, device=out.device) // c["C"]
            hidden = pos_k[None] > pos_q[:, None]
            if c["R"] >= 0:
                hidden |= pos_k[None] < pos_q[:, None] - c["R"]
        else:
            keys, values, hidden = s["k"][b, :, :nk], s["v"][b, :, :nk], None
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            q, k, v = (x.detach().double().requires_grad_(train) for x in (s["q"][b, heads, :nq], keys[h], values[h]))
            x = (q @ k.T) / math.sqrt(D)
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            o = torch.softmax(x, -1) @ v
            out[b, heads, :nq] = o.detach()
            lse[b, heads, :nq] = torch.logsumexp(x.detach(), -1) / math.log(2)
            if train:
                g = torch.autograd.grad(o, (q, k, v), s["d_o"][b, heads, :nq].double())
                grads[0][b, heads, :nq] = g[0]
                grads[1][b, h, :nk], grads[2][b, h, :nk] = g[1], g[2]
    if train:
        return (out, *grads)
    return (out, lse) if c["lse"] else out
