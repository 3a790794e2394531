"""Host-side checks of norms and rotation, trees of drafted tokens and keeping that need no GPU: the C ABI refuses bad arguments
before any device work, the public functions refuse them by name, and the references agree with the oracle."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from kv_attention import _lib, ops
from oracle import kv_oracle
from paged_attention import paged_append_rope, paged_keep, paged_tree_attention, paged_tree_attention_reference
from qk_norm_rope import qk_norm_rope, qk_norm_rope_reference


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def _buffer():
    buf = ctypes.create_string_buffer(256)
    return buf, (ctypes.addressof(buf) + 15) & ~15


def test_rope_codes(lib):
    buf, p = _buffer()
    st, two = _strides(8 * 64, 8 * 64, 64, 1), _strides(3, 1)
    base = dict(q=p, k=p, cos=p, sin=p, cs=32, ss=32, wq=p, wk=p, pos=None, ps=two, qo=p, ko=p, qs=st, ks=st, B=1, Hq=2, Hkv=1, T=8, D=64, rot=64,
                rows=8, eps=1e-6, dtype=2)

    def forward(**kw):
        a = dict(base, **kw)
        return lib.kv_qk_norm_rope(a["q"], a["k"], a["cos"], a["sin"], a["cs"], a["ss"], a["wq"], a["wk"], 0, None, 0, a["pos"], a["ps"], a["qo"],
                                   a["ko"], a["qs"], a["ks"], a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["rot"], a["rows"], 0, a["eps"],
                                   a["dtype"], None)

    def backward(**kw):
        a = {**base, "dwq": p, "dwk": p, "ws": p, "bytes": 1 << 30, "g": p, "gs": st, **kw}
        return lib.kv_qk_norm_rope_backward(a["q"], a["k"], a["g"], a["g"], a["cos"], a["sin"], a["cs"], a["ss"], a["wq"], a["wk"], 0, None, 0,
                                            a["pos"], a["ps"], a["qo"], a["ko"], a["dwq"], a["dwk"], a["ws"], a["bytes"], a["qs"], a["ks"], a["gs"],
                                            a["gs"], a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["rot"], a["rows"], 0, a["eps"], a["dtype"], None)

    def append(**kw):
        a = dict(base, kp=p, vp=p, table=p, lens=p, v=p, kps=st, vps=st, N=4, page=8, W=3)
        a.update(kw)
        return lib.kv_paged_append_rope(a["q"], a["k"], a["v"], a["qo"], a["kp"], a["vp"], a["table"], 3, a["lens"], 1, None, 0, a["cos"], a["sin"],
                                        a["cs"], a["ss"], a["wq"], a["wk"], 0, a["pos"], a["ps"], a["qs"], a["ks"], a["ks"], a["kps"], a["vps"],
                                        a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["N"], a["page"], a["W"], a["rot"], a["rows"], 0, a["eps"],
                                        a["dtype"], None)

    for f in (forward, backward, append):
        assert f(dtype=3) == -1 and f(D=48) == -2
        assert f(B=-1) == -3 and f(T=-1) == -3 and f(Hq=-1) == -3 and f(rows=-1) == -3
        assert f(rot=8) == -3 and f(rot=24) == -3 and f(rot=80) == -3 and f(rot=0) == -3
        assert f(eps=-1.0) == -3 and f(eps=float("nan")) == -3 and f(eps=float("inf")) == -3 and f(eps=0.0) == -3   # weights without norms
        assert f(q=None) == -3 and f(k=None) == -3 and f(qo=None) == -3 and f(cos=None) == -3 and f(sin=None) == -3
        assert f(q=p + 2) == -4 and f(qs=_strides(512, 512, 60, 1)) == -4 and f(ks=_strides(512, 512, 64, 2)) == -4 and f(cos=p + 4) == -4
        assert f(cs=33) == -4 and f(ss=-32) == -4 and f(wq=p + 2) == -4
        assert f(pos=p, ps=None) == -3
        assert f(B=1 << 20, T=1 << 12) == -5 and f(Hq=40000) == -5
    for f in (forward, append):
        assert f(B=0) == 0 and f(T=0) == 0
    for f in (forward, backward):
        assert f(ko=None) == -3
    assert backward(g=None) == -3 and backward(g=p + 4) == -4 and backward(dwq=p + 4, dwk=None) == -4
    assert backward(wq=None, dwq=p, dwk=None) == -3
    need = lib.kv_qk_norm_rope_backward_workspace(1, 2, 1, 8, 64, 2)
    assert need > 0 and backward(bytes=need - 1) == -6 and backward(ws=None) == -6 and backward(ws=p + 4) == -4
    assert backward(dwq=None, dwk=None, B=0) == 0
    assert append(lens=None) == -3 and append(table=None) == -3 and append(v=None) == -3 and append(kp=p + 8) == -4
    assert append(kps=_strides(512, 0, 64, 1), Hkv=2, Hq=2) == -4 and append(vps=_strides(0, 512, 64, 1)) == -4
    assert append(page=0) == -3 and append(N=-1) == -3 and append(W=-1) == -3 and append(W=1 << 21, page=1 << 10) == -5
    assert lib.kv_qk_norm_rope_backward_workspace(1, 2, 1, 8, 63, 2) == -2 and lib.kv_qk_norm_rope_backward_workspace(0, 2, 1, 8, 64, 2) == 0
    assert lib.kv_qk_norm_rope_backward_workspace(64, 64, 64, 1 << 16, 256, 0) <= 1 << 24   # sums of workgroups, not of tokens


def test_rope_without_heads(lib):
    """No query or key heads, or neither: nothing to do, whatever else stands there."""
    def call(B, T):
        return lib.kv_qk_norm_rope_backward(None, None, None, None, None, None, 0, 0, None, None, 0, None, 0, None, None, None, None, None, None,
                                            None, 0, None, None, None, None, B, 0, 0, T, 64, 64, 0, 0, 1e-6, 2, None)

    for B, T in ((1, 8), (0, 8), (3, 0)):
        assert call(B, T) == 0
        assert lib.kv_qk_norm_rope_backward_workspace(B, 0, 0, T, 64, 2) == 0
        assert lib.kv_qk_norm_rope(None, None, None, None, 0, 0, None, None, 0, None, 0, None, None, None, None, None, None, B, 0, 0, T, 64, 64, 0, 0,
                                   1e-6, 2, None) == 0


def test_tree_and_keep_codes(lib):
    buf, p = _buffer()
    st, three = _strides(8 * 64, 8 * 64, 64, 1), _strides(1, 1, 1)
    base = dict(q=p, k=p, table=p, lens=p, tree=p, ts=three, o=p, ws=None, bytes=0, qs=st, ks=st, B=1, Hq=2, Hkv=1, T=1, D=64, N=4, page=8, W=3,
                scale=0.1, dtype=1)

    def tree(**kw):
        a = dict(base, **kw)
        return lib.kv_paged_tree_forward(a["q"], a["k"], a["k"], a["table"], 3, a["lens"], 1, None, 0, a["tree"], a["ts"], a["o"], None, a["ws"],
                                         a["bytes"], a["qs"], a["ks"], a["ks"], a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["N"], a["page"],
                                         a["W"], a["scale"], a["dtype"], None)

    def keep(**kw):
        a = dict(base, first=p, kept=p, es=_strides(3, 1), M=2)
        a.update(kw)
        return lib.kv_paged_keep(a["k"], a["k"], a["table"], 3, a["first"], 1, a["kept"], a["es"], a["ks"], a["ks"], a["B"], a["Hkv"], a["M"], a["D"],
                                 a["N"], a["page"], a["W"], a["dtype"], None)

    for f in (tree, keep):
        assert f(dtype=7) == -1 and f(D=17) == -2
        assert f(page=0) == -3 and f(W=-1) == -3 and f(N=-1) == -3 and f(B=-2) == -3
        assert f(table=None) == -3 and f(k=None) == -3
        assert f(k=p + 2) == -4 and f(ks=_strides(512, 512, 60, 1)) == -4 and f(ks=_strides(512, 512, 64, 2)) == -4
        assert f(W=1 << 21, page=1 << 10) == -5
        assert f(B=0) == 0
    assert tree(T=-1) == -3 and tree(Hq=3, Hkv=2) == -3 and tree(o=None) == -3 and tree(tree=None) == -3 and tree(ts=None) == -3
    assert tree(lens=None) == -3 and tree(q=None) == -3 and tree(T=0) == 0
    for scale in (3e38, float("nan"), float("inf")):
        assert tree(scale=scale) == -3
    need = lib.kv_paged_tree_forward_workspace(1, 2, 1, 1, 64, 8, 1000, 1)
    assert need > 0 and tree(W=1000, ws=p, bytes=need - 1) == -6 and tree(W=1000, ws=p + 4, bytes=need) == -4
    assert tree(B=1 << 24, Hq=1) == -5
    assert keep(first=None) == -3 and keep(kept=None) == -3 and keep(es=None) == -3 and keep(M=-1) == -3
    assert keep(M=0) == 0 and keep(N=0) == 0 and keep(W=0) == 0
    assert keep(ks=_strides(512, 0, 64, 1), Hkv=2) == -4 and keep(ks=_strides(0, 512, 64, 1)) == -4


def test_tree_parts_stay_small(lib):
    for B, Hq, T in ((8, 64, 2048), (128, 64, 4), (1, 8, 1), (64, 32, 64)):
        assert 0 <= lib.kv_paged_tree_forward_workspace(B, Hq, 8, T, 128, 16, 4096, 2) <= 1 << 28


def _rope(**kw):
    a = dict(q=torch.zeros(2, 4, 5, 64), k=torch.zeros(2, 2, 5, 64), cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), q_weight=None, k_weight=None,
             lens=None, positions=None, eps=1e-6)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 4, 64)), dict(k=torch.zeros(2, 2, 6, 64)), dict(k=torch.zeros(3, 2, 5, 64)), dict(k=torch.zeros(2, 2, 5, 32)),
    dict(k=torch.zeros(2, 2, 5, 64).half()), dict(q=torch.zeros(2, 4, 5, 64).double(), k=torch.zeros(2, 2, 5, 64).double()),
    dict(k=torch.zeros(2, 0, 5, 64)), dict(k=torch.zeros(2, 2, 5, 64, device="meta")),
    dict(cos=torch.zeros(9, 32).half()), dict(cos=torch.zeros(9)), dict(cos=torch.zeros(8, 32)), dict(cos=torch.zeros(9, 32, device="meta")),
    dict(cos=torch.zeros(9, 4), sin=torch.zeros(9, 4)), dict(cos=torch.zeros(9, 12), sin=torch.zeros(9, 12)),
    dict(cos=torch.zeros(9, 40), sin=torch.zeros(9, 40)), dict(cos=torch.zeros(9, 0), sin=torch.zeros(9, 0)),
    dict(q_weight=torch.ones(32)), dict(q_weight=torch.ones(1, 64)), dict(k_weight=torch.ones(64).half()), dict(k_weight=torch.ones(64).double()),
    dict(q_weight=torch.ones(64, device="meta")), dict(eps=0.0), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e-60),
    dict(eps=None, q_weight=torch.ones(64)), dict(lens=torch.zeros(2)), dict(lens=torch.zeros(3, dtype=torch.int32)),
    dict(positions=torch.zeros(2, 5)), dict(positions=torch.zeros(5, dtype=torch.int32)), dict(positions=torch.zeros(1, 5, dtype=torch.int32)),
    dict(positions=torch.zeros(2, 5, dtype=torch.int64)), dict(positions=torch.zeros(2, 5, dtype=torch.int32, device="meta")),
])
def test_rope_refusals(kw):
    with pytest.raises(AssertionError):
        ops._validate_rope(*_rope(**kw))


def test_rope_accepts():
    ops._validate_rope(*_rope())
    ops._validate_rope(*_rope(eps=None))
    half = {n: torch.zeros(2, h, 5, 64).half() for n, h in (("q", 3), ("k", 2))}
    ops._validate_rope(*_rope(**half, q_weight=torch.ones(64), k_weight=torch.ones(64), positions=torch.zeros(2, 5, dtype=torch.int32)))
    with pytest.raises(AssertionError):
        ops._validate_rope(*_rope(**half, q_weight=torch.ones(64), k_weight=torch.ones(64).half()))
    with pytest.raises(AssertionError):
        ops._validate_rope(*_rope(), torch.zeros(2, 4, 5, 64), torch.zeros(2, 4, 5, 64))


def _append(**kw):
    a = dict(q=torch.zeros(2, 4, 5, 64), k=torch.zeros(2, 2, 5, 64), v=torch.zeros(2, 2, 5, 64), k_pages=torch.zeros(9, 2, 16, 64),
             v_pages=torch.zeros(9, 2, 16, 64), page_table=torch.zeros(2, 5, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32),
             cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), q_weight=None, k_weight=None, new_lens=None, positions=None, eps=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 4, 6, 64)), dict(q=torch.zeros(2, 3, 5, 64)), dict(v=torch.zeros(2, 2, 6, 64)), dict(v=torch.zeros(2, 2, 5, 64).half()),
    dict(k=torch.zeros(2, 4, 5, 64), v=torch.zeros(2, 4, 5, 64)), dict(k_pages=torch.zeros(9, 2, 16, 66)[..., :64]), dict(lens=None),
    dict(new_lens=torch.zeros(3, dtype=torch.int32)), dict(page_table=torch.zeros(3, 5, dtype=torch.int32)), dict(cos=torch.zeros(9, 16)),
    dict(q_weight=torch.ones(64)), dict(eps=0.0), dict(positions=torch.zeros(2, 4, dtype=torch.int32)),
])
def test_append_rope_refusals(kw):
    ops._validate_append_rope(*_append())
    with pytest.raises(AssertionError):
        ops._validate_append_rope(*_append(**kw))


@pytest.mark.parametrize("kw", [
    dict(tree=torch.ones(3, 3)), dict(tree=torch.ones(4, 4, dtype=torch.bool)), dict(tree=torch.ones(3, 4, dtype=torch.bool)),
    dict(tree=torch.ones(3, 3, 3, dtype=torch.bool)), dict(tree=torch.ones(1, 3, 3, dtype=torch.bool)), dict(tree=torch.ones(3, dtype=torch.bool)),
    dict(tree=torch.ones(3, 3, dtype=torch.bool, device="meta")), dict(sm_scale=1e39), dict(lens=None), dict(q=torch.zeros(2, 3, 3, 64)),
    dict(k_pages=torch.zeros(1, 2, 16, 64).expand(9, 2, 16, 64)), dict(new_lens=torch.zeros(2)),
])
def test_tree_refusals(kw):
    a = dict(q=torch.zeros(2, 4, 3, 64), k_pages=torch.zeros(9, 2, 16, 64), v_pages=torch.zeros(9, 2, 16, 64),
             page_table=torch.zeros(2, 5, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32), tree=torch.ones(3, 3, dtype=torch.bool),
             sm_scale=0.1, new_lens=None)
    ops._validate_tree(*a.values())
    ops._validate_tree(*{**a, "tree": torch.ones(2, 3, 3, dtype=torch.bool)}.values())
    with pytest.raises(AssertionError):
        ops._validate_tree(*{**a, **kw}.values())


@pytest.mark.parametrize("kw", [
    dict(first=torch.zeros(2)), dict(first=torch.zeros(3, dtype=torch.int32)), dict(kept=torch.zeros(2, 4)), dict(kept=torch.zeros(2, dtype=torch.int32)),
    dict(kept=torch.zeros(3, 4, dtype=torch.int32)), dict(v_pages=torch.zeros(9, 2, 16, 32)), dict(v_pages=torch.zeros(9, 2, 16, 64).half()),
    dict(k_pages=torch.zeros(9, 2, 16, 64).double(), v_pages=torch.zeros(9, 2, 16, 64).double()), dict(page_table=torch.zeros(2, 5)),
    dict(page_table=torch.zeros(10, dtype=torch.int32)), dict(k_pages=torch.zeros(9, 2, 16, 128)[..., ::2]),
    dict(first=torch.zeros(2, dtype=torch.int32, device="meta")),
])
def test_keep_refusals(kw):
    a = dict(k_pages=torch.zeros(9, 2, 16, 64), v_pages=torch.zeros(9, 2, 16, 64), page_table=torch.zeros(2, 5, dtype=torch.int32),
             first=torch.zeros(2, dtype=torch.int32), kept=torch.zeros(2, 4, dtype=torch.int32))
    ops._validate_keep(*a.values())
    with pytest.raises(AssertionError):
        ops._validate_keep(*{**a, **kw}.values())


def _meta(*shape, **kw):
    return torch.randn(*shape, device="meta", **kw)


def test_autograd_surface():
    q, k, w = _meta(2, 4, 5, 64, requires_grad=True), _meta(2, 2, 5, 64, requires_grad=True), _meta(64, requires_grad=True)
    cos, sin = _meta(9, 32), _meta(9, 32)
    out = qk_norm_rope(q, k, cos, sin, w, w)
    assert [t.shape for t in out] == [q.shape, k.shape] and all(t.requires_grad for t in out)
    grads = torch.autograd.grad([t.sum() for t in out], (q, k, w), create_graph=True)
    assert [g.shape for g in grads] == [q.shape, k.shape, w.shape]
    with pytest.raises(RuntimeError, match="double backward"):
        grads[0].sum().backward()
    only = qk_norm_rope(q.detach(), k.detach(), cos, sin, None, w)
    assert torch.autograd.grad(only[1].sum(), w)[0].shape == (64,)
    with torch.no_grad():
        assert not qk_norm_rope(q, k, cos, sin, w, w)[0].requires_grad
    with pytest.raises(RuntimeError, match="detach"):
        qk_norm_rope(q, k, _meta(9, 32, requires_grad=True), sin)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        qk_norm_rope(forward_ad.make_dual(_meta(2, 4, 5, 64), _meta(2, 4, 5, 64)), k.detach(), cos, sin)
    assert qk_norm_rope(q, k, cos, sin, eps=1)[0].shape == q.shape   # converted

    table, lens, pages = torch.zeros(2, 5, dtype=torch.int32, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta"), _meta(9, 2, 16, 64)
    tree, kept = torch.ones(5, 5, dtype=torch.bool, device="meta"), torch.zeros(2, 3, dtype=torch.int32, device="meta")
    o, lse = paged_tree_attention(q.detach(), pages, pages, table, lens, tree, return_lse=True)
    assert o.shape == q.shape and lse.shape == (2, 4, 5) and not o.requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula"):
        paged_tree_attention(q, pages, pages, table, lens, tree).sum().backward()
    with pytest.raises(RuntimeError, match="records no gradient"):
        paged_append_rope(q.detach(), k, k.detach(), pages, pages, table, lens, cos, sin)
    with pytest.raises(RuntimeError, match="records no gradient"):
        paged_append_rope(q.detach(), k.detach(), k.detach(), pages, pages, table, lens, cos, sin, w, eps=1e-6)
    with pytest.raises(RuntimeError, match="records no gradient"):
        paged_keep(_meta(9, 2, 16, 64, requires_grad=True), pages, table, lens, kept)
    with torch.no_grad():
        assert paged_append_rope(q, k, k, pages, pages, table, lens, cos, sin, w, eps=1e-6).shape == q.shape
        assert paged_keep(pages, pages, table, lens, kept) is None


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("eps", [None, 1e-3])
def test_references_agree_with_the_oracle(interleaved, eps):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 4, 6, 32, generator=g), torch.randn(2, 2, 6, 32, generator=g)
    w = None if eps is None else 1 + 0.2 * torch.randn(32, generator=g)
    angle = torch.arange(6)[:, None] * torch.rand(8, generator=g)
    cos, sin = angle.cos(), angle.sin()
    leaves = [t.double().requires_grad_() for t in (q, k)]
    out = qk_norm_rope_reference(*leaves, cos.double(), sin.double(), w, w, eps=eps, interleaved=interleaved)
    up = [torch.randn(t.shape, generator=g) for t in out]
    grads = torch.autograd.grad(out, leaves, [t.double() for t in up])
    for x, o, dx, u in zip((q, k), out, grads, up):
        want = kv_oracle.rope_rows(x, cos, sin, w, eps, interleaved, u)
        assert (o - want["out"][0]).abs().max() < 1e-12 and (dx - want["dx"][0]).abs().max() < 1e-12
    # a rotation keeps the length of every pair, and the angle between two tokens is that of their distance
    turned = kv_oracle.rope_rows(q, cos, sin, None, None, interleaved)[0]
    assert (turned.norm(dim=-1) - q.double().norm(dim=-1)).abs().max() < 1e-5
    x = q[:1, :1, :1].expand(1, 1, 6, 32)
    turned = kv_oracle.rope_rows(x, cos, sin, None, None, interleaved)[0][0, 0]
    dots = turned @ turned.T
    assert (dots.diagonal(1) - dots[0, 1]).abs().max() < 1e-5


def test_reference_of_trees_agrees_with_the_oracle():
    g = torch.Generator().manual_seed(2)
    q = torch.randn(3, 4, 6, 16, generator=g)
    pages = [torch.randn(7, 2, 4, 16, generator=g) for _ in range(2)]
    table = torch.tensor([[6, 2, -1, 5], [0, 9, 1, 3], [1, 2, 3, 4]], dtype=torch.int32)
    tree = torch.rand(3, 6, 6, generator=g) < 0.5
    for lens, new in (([15, 3, 6], None), ([16, 6, 0], [2, 6, 5]), ([40, -1, 4], [9, -1, 6])):
        lens, new = torch.tensor(lens, dtype=torch.int32), None if new is None else torch.tensor(new, dtype=torch.int32)
        for mask in (tree, tree[0]):
            got, _ = paged_tree_attention_reference(q.double(), *[p.double() for p in pages], table, lens, mask, new_lens=new)
            assert (got - kv_oracle.tree(q, *pages, table, lens, mask, None, new)["o"][0]).abs().max() < 1e-12


def test_bounds_catch_a_planted_mistake():
    """A neighbour's angle, a weight left out, one token too many in a tree: all outside the bounds."""
    g = torch.Generator().manual_seed(3)
    x, up = (torch.randn(20, 64, generator=g).bfloat16() for _ in range(2))
    angle = torch.arange(21)[:, None] * 10000.0 ** (-torch.arange(32) / 32)
    cos, sin = angle.cos(), angle.sin()
    w = 1 + 0.2 * torch.randn(64, generator=g)
    good = kv_oracle.rope_rows(x, cos[:20], sin[:20], w, 1e-6, False, up)
    late = kv_oracle.rope_rows(x, cos[1:], sin[1:], w, 1e-6, False, up)
    plain = kv_oracle.rope_rows(x, cos[:20], sin[:20], torch.ones(64), 1e-6, False, up)
    for name in ("out", "dx", "dw"):
        for other in (late, plain) if name != "dw" else (late,):
            with pytest.raises(AssertionError):
                kv_oracle.assert_within(name, other[name][0], good[name])
    q = torch.randn(1, 2, 5, 64, generator=g).half()
    pages = [torch.randn(9, 2, 16, 64, generator=g).half() for _ in range(2)]
    table, lens = torch.arange(9, dtype=torch.int32)[None], torch.tensor([100], dtype=torch.int32)
    tree = torch.eye(5, dtype=torch.bool)
    good = kv_oracle.tree(q, *pages, table, lens, tree)
    tree[3, 1] = True
    other = kv_oracle.tree(q, *pages, table, lens, tree)
    for name in ("o", "lse"):
        with pytest.raises(AssertionError):
            kv_oracle.assert_within(name, other[name][0], good[name])
