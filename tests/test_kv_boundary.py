"""Host-side checks of cross attention and attention over pages that need no GPU: the C ABI exports what its header declares and
refuses bad arguments before any device work; the public functions refuse bad arguments, and name the condition."""
import ctypes
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from cross_attention import cross_attention, cross_attention_reference
from kv_attention import _lib, ops
from oracle import kv_oracle
from paged_attention import paged_append, paged_attention, paged_attention_reference

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_header_symbols_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "kv_attention.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(kv_[a-z_]+)\s*\(", text)))
    assert names == sorted(_lib.SIGNATURES)
    for n in names:
        assert getattr(lib, n) is not None
    for n, args in re.findall(r"\b(kv_[a-z_]+)\s*\(([^)]*)\)", text):
        assert len(args.split(",")) == len(_lib.SIGNATURES[n]), n
    for code in range(-6, 0):
        assert len(lib.kv_error_string(code)) > 10


def _strides(*s):
    return (ctypes.c_int64 * 4)(*s)


def _buffer():
    buf = ctypes.create_string_buffer(256)
    return buf, (ctypes.addressof(buf) + 15) & ~15


def test_cross_codes(lib):
    buf, p = _buffer()
    st = _strides(8 * 64, 8 * 64, 64, 1)
    base = dict(q=p, k=p, o=p, ws=None, bytes=0, qs=st, ks=st, B=1, Hq=2, Hkv=1, Tq=8, Tk=8, D=64, dtype=2)

    def forward(**kw):
        a = dict(base, **kw)
        return lib.kv_cross_forward(a["q"], a["k"], a["k"], None, 0, None, 0, a["o"], None, a["ws"], a["bytes"], a["qs"], a["ks"], a["ks"],
                                    a["B"], a["Hq"], a["Hkv"], a["Tq"], a["Tk"], a["D"], 0.1, a["dtype"], None)

    def backward(**kw):
        a = dict(base, **kw)
        return lib.kv_cross_backward(a["q"], a["k"], a["k"], None, 0, None, 0, p, p, a.get("lse", p), a["o"], p, p, a["ws"], a["bytes"],
                                     a["qs"], a["ks"], a["ks"], st, st, a["B"], a["Hq"], a["Hkv"], a["Tq"], a["Tk"], a["D"], 0.1,
                                     a["dtype"], None)

    for f in (forward, backward):
        assert f(dtype=3) == -1 and f(dtype=-1) == -1
        assert f(D=48) == -2 and f(D=512) == -2
        assert f(Hq=3, Hkv=2) == -3 and f(Hkv=0) == -3 and f(B=-1) == -3 and f(Tk=-1) == -3 and f(Tq=-1) == -3
        assert f(q=None) == -3 and f(o=None) == -3 and f(k=None) == -3
        assert f(q=p + 2) == -4 and f(o=p + 8) == -4
        assert f(qs=_strides(512, 512, 64, 2)) == -4 and f(ks=_strides(512, 512, 63, 1)) == -4
        assert f(ks=_strides(512, 512, 0, 1)) == -4 and f(ks=_strides(512, 512, -64, 1)) == -4 and f(ks=_strides(-8, 512, 64, 1)) == -4
        assert f(ks=_strides(512, 512, 1 << 21, 1)) == -5        # 1032 rows of 4 MiB
        assert f(Hq=1 << 20, Hkv=1, Tq=1 << 12) == -5            # rows beyond 31 bits
        assert f(B=0) == 0
    assert forward(Tq=0) == 0
    assert backward(lse=None) == -3
    assert backward() == -6 and backward(ws=p, bytes=16) == -6   # the backward always has a workspace
    need = lib.kv_cross_forward_workspace(1, 1, 1, 40, 10000, 64, 2)
    assert need > 0 and forward(Hq=1, Tq=40, Tk=10000, ws=p, bytes=need - 1) == -6
    assert forward(Hq=1, Tq=40, Tk=10000, ws=None, bytes=need) == -6 and forward(Hq=1, Tq=40, Tk=10000, ws=p + 4, bytes=need) == -4
    assert lib.kv_cross_forward_workspace(1, 1, 1, 40, 10000, 63, 2) == -2
    assert lib.kv_cross_backward_workspace(1, 2, 3, 40, 10000, 64, 2) == -3
    assert lib.kv_cross_forward_workspace(64, 16, 16, 500, 1500, 64, 2) == 0


def test_paged_codes(lib):
    buf, p = _buffer()
    st = _strides(8 * 64, 8 * 64, 64, 1)
    base = dict(q=p, k=p, table=p, lens=p, o=p, qs=st, ks=st, B=1, Hq=2, Hkv=1, T=1, D=64, N=4, page=8, W=3, C=1, R=9, dtype=1)

    def forward(**kw):
        a = dict(base, **kw)
        return lib.kv_paged_forward(a["q"], a["k"], a["k"], a["table"], 3, a["lens"], 1, None, 0, a["o"], None, a.get("ws"), a.get("bytes", 0),
                                    a["qs"], a["ks"], a["ks"], a["B"], a["Hq"], a["Hkv"], a["T"], a["D"], a["N"], a["page"], a["W"], a["C"],
                                    a["R"], 0.1, a["dtype"], None)

    def append(**kw):
        a = dict(base, **kw)
        return lib.kv_paged_append(a["q"], a["q"], a["k"], a["k"], a["table"], 3, a["lens"], 1, None, 0, a["qs"], a["qs"], a["ks"], a["ks"],
                                   a["B"], a["Hq"], a["T"], a["D"], a["N"], a["page"], a["W"], a["dtype"], None)

    for f in (forward, append):
        assert f(dtype=7) == -1 and f(D=17) == -2
        assert f(page=0) == -3 and f(W=-1) == -3 and f(N=-1) == -3 and f(T=-1) == -3 and f(B=-2) == -3
        assert f(lens=None) == -3 and f(table=None) == -3 and f(q=None) == -3 and f(k=None) == -3
        assert f(k=p + 2) == -4 and f(ks=_strides(512, 512, 60, 1)) == -4 and f(ks=_strides(512, 512, 64, 2)) == -4
        assert f(W=1 << 21, page=1 << 10) == -5                  # positions beyond 2^30
        assert f(B=0) == 0 and f(T=0) == 0
    assert forward(Hq=3, Hkv=2) == -3 and forward(C=0) == -3 and forward(R=-1) == -3 and forward(o=None) == -3
    assert append(B=1 << 15, T=1 << 15) == -5
    assert append(N=0) == 0 and append(W=0) == 0
    assert append(ks=_strides(512, 0, 64, 1)) == -4 and append(ks=_strides(0, 512, 64, 1)) == -4   # two heads, or two pages, in one place
    need = lib.kv_paged_forward_workspace(1, 2, 1, 1, 64, 8, 1000, 1, 2 ** 31 - 1, 1)
    assert need > 0 and forward(W=1000, R=2 ** 31 - 1, ws=p, bytes=need - 1) == -6
    assert lib.kv_paged_forward_workspace(1, 2, 1, 1, 64, 8, 1000, 1, 100, 1) == 0       # a short window is not divided


@pytest.mark.parametrize("B,T,G,page,width,C,R", [(2, 1, 1, 16, 4000, 1, 2 ** 31 - 1), (1, 40, 3, 7, 900, 13, 60), (3, 5, 40, 1, 3000, 1, 900),
                                                  (1, 33, 1, 64, 100, 1000, 3), (1, 64, 8, 32, 200, 64, 31), (1, 2, 16, 16, 500, 17, 200)])
def test_shares_cover_every_window(lib, B, T, G, page, width, C, R):
    """The shares that the host counts reach over the tiles that any 32 rows see together, for every length."""
    most, D = width * page, 64
    bytes_ = lib.kv_paged_forward_workspace(B, 2 * G, 2, T, D, page, width, C, R, 1)
    splits = bytes_ // (B * 2 * G * T * (D + 2) * 4) if bytes_ else 1
    tokens = min(T, 31 // G + 2)
    tiles = 0
    for L in sorted({*range(1, 200), *range(max(1, most - 300), most + 1)} & set(range(1, most + 1))):
        for r0 in range(0, G * T, 32):
            at = [max(0, min(L - 1, L - T + r // G)) for r in (r0, min(r0 + 31, G * T - 1))]
            lo = max(at[0] // C - R, 0) * C
            hi = min((at[1] // C + 1) * C, L)
            tiles = max(tiles, -(-hi // 32) - lo // 32)
    n = min(-(-most // 32), -(-min(most, (R + -(-(tokens - 1) // C) + 1) * C) // 32) + 1)
    units = B * 2 * -(-G * T // 32)
    share = max(4, -(-units * n // 256))
    if n <= 32 or (2 * share >= n and n <= 64):   # (float16 at head dimension 64)
        share = n
    else:
        share = max(min(32 if share > 32 and units * -(-n // 32) >= 1024 else share, 128), -(-n // 256))
    assert splits == -(-n // share) and tiles <= splits * share
    assert bytes_ <= 1 << 28


def test_parts_stay_small(lib):
    """A long chunk of many sequences does not ask for a workspace of gigabytes."""
    for B, Hq, T in ((8, 64, 2048), (128, 64, 4), (1, 8, 1), (512, 128, 1)):
        assert 0 <= lib.kv_paged_forward_workspace(B, Hq, 8, T, 128, 16, 4096, 1, 2 ** 31 - 1, 2) <= 1 << 28
    assert lib.kv_paged_forward_workspace(64, 64, 8, 1, 128, 16, 4096, 1, 2 ** 31 - 1, 2) > 0   # and few rows are still divided


@pytest.mark.parametrize("dtype,es", [(0, 4), (1, 2)])
def test_cross_parts_stay_small(lib, dtype, es):
    """Parts of divided runs: a few times the rows of a GPU full of workgroups, however long the other side is."""
    for D in (16, 64, 128, 256):
        for B, Hq, Hkv, Tq, Tk in ((1, 1, 1, 100, 1 << 20), (3, 16, 4, 1424, 14631), (1, 8, 8, 4096, 1 << 20), (1, 1, 1, 1 << 20, 100),
                                   (64, 16, 16, 40, 9000), (13, 16, 1, 3974, 15)):
            most = 9 * 256 * 128 * (D + 2) * 4
            assert 0 <= lib.kv_cross_forward_workspace(B, Hq, Hkv, Tq, Tk, D, dtype) <= most
            stats = 2 * (B * Hq * Tq * 4 + 256)
            assert 0 < lib.kv_cross_backward_workspace(B, Hq, Hkv, Tq, Tk, D, dtype) <= stats + most


def _cross(dtype=torch.float32, **kw):
    a = dict(q=torch.zeros(2, 4, 5, 64, dtype=dtype), k=torch.zeros(2, 2, 7, 64, dtype=dtype), v=torch.zeros(2, 2, 7, 64, dtype=dtype),
             lens=None, q_lens=None, sm_scale=0.1)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 4, 64)), dict(k=torch.zeros(2, 2, 7, 32)), dict(k=torch.zeros(2, 2, 8, 64)), dict(v=torch.zeros(2, 1, 7, 64)),
    dict(q=torch.zeros(2, 3, 5, 64)), dict(q=torch.zeros(3, 4, 5, 64)), dict(q=torch.zeros(2, 4, 5, 64, dtype=torch.float16)),
    dict(lens=torch.zeros(2, dtype=torch.int64)), dict(lens=torch.zeros(3, dtype=torch.int32)), dict(q_lens=torch.zeros(2, 1, dtype=torch.int32)),
    dict(q_lens=torch.zeros(2, dtype=torch.int32, device="meta")), dict(sm_scale=float("nan")), dict(sm_scale=float("inf")),
    dict(k=torch.zeros(2, 0, 7, 64), v=torch.zeros(2, 0, 7, 64)),
])
def test_cross_refusals(kw):
    with pytest.raises(AssertionError):
        ops._validate_cross(*_cross(**kw))


def test_cross_refuses_types_and_head_dims():
    for bad in (_cross(torch.float64), tuple(t[..., :48] if torch.is_tensor(t) else t for t in _cross())):
        with pytest.raises(AssertionError):
            ops._validate_cross(*bad)
    ops._validate_cross(*_cross(lens=torch.zeros(2, dtype=torch.int32)))
    with pytest.raises(AssertionError):
        ops._validate_cross(*_cross(), torch.zeros(2, 4, 5, 32), torch.zeros(2, 4, 5, 64))


def _paged(**kw):
    a = dict(q=torch.zeros(2, 4, 1, 64), k_pages=torch.zeros(9, 2, 16, 64), v_pages=torch.zeros(9, 2, 16, 64),
             page_table=torch.zeros(2, 5, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32), context_size=1, back_contexts=0,
             sm_scale=0.1, new_lens=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw", [
    dict(k_pages=torch.zeros(9, 2, 16, 65)[..., 1:]), dict(v_pages=torch.zeros(9, 2, 16, 66)[..., :64]),
    dict(k_pages=torch.zeros(9, 2, 16, 128)[..., ::2]), dict(k_pages=torch.zeros(1, 2, 16, 64).expand(9, 2, 16, 64)),
    dict(k_pages=torch.zeros(8, 2, 16, 64)), dict(page_table=torch.zeros(2, 5)), dict(page_table=torch.zeros(3, 5, dtype=torch.int32)),
    dict(page_table=torch.zeros(10, dtype=torch.int32)), dict(lens=None), dict(lens=torch.zeros(2)), dict(new_lens=torch.zeros(1, dtype=torch.int32)),
    dict(context_size=0), dict(back_contexts=-1), dict(sm_scale=float("inf")), dict(q=torch.zeros(2, 3, 1, 64)),
    dict(q=torch.zeros(2, 4, 1, 32)), dict(page_table=torch.zeros(2, 1, dtype=torch.int32).expand(2, (1 << 26) + 1)),
])
def test_paged_refusals(kw):
    with pytest.raises(AssertionError):
        ops._validate_paged(*_paged(**kw))


def test_append_refusals():
    ok = dict(k=torch.zeros(2, 2, 3, 64), v=torch.zeros(2, 2, 3, 64), k_pages=torch.zeros(9, 2, 16, 64), v_pages=torch.zeros(9, 2, 16, 64),
              page_table=torch.zeros(2, 5, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32), new_lens=None)
    ops._validate_append(*ok.values())
    for kw in (dict(k=torch.zeros(2, 4, 3, 64), v=torch.zeros(2, 4, 3, 64)), dict(v=torch.zeros(2, 2, 2, 64)), dict(v=torch.zeros(2, 2, 3, 64).half()),
               dict(lens=None), dict(new_lens=torch.zeros(2))):
        with pytest.raises(AssertionError):
            ops._validate_append(*{**ok, **kw}.values())


def _meta(*shape, **kw):
    return torch.randn(*shape, device="meta", **kw)


def test_autograd_surface():
    q, k, v = _meta(2, 4, 5, 64, requires_grad=True), _meta(2, 2, 7, 64, requires_grad=True), _meta(2, 2, 7, 64)
    o, lse = cross_attention(q, k, v, return_lse=True)
    assert o.requires_grad and not lse.requires_grad and lse.shape == (2, 4, 5)
    gq, gk = torch.autograd.grad(o.sum(), (q, k), create_graph=True)
    assert gq.shape == q.shape and gk.shape == k.shape
    with pytest.raises(RuntimeError, match="double backward"):
        gq.sum().backward()
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        cross_attention(forward_ad.make_dual(_meta(2, 4, 5, 64), _meta(2, 4, 5, 64)), k.detach(), v)
    with torch.no_grad():
        assert not cross_attention(q, k, v).requires_grad

    table, lens = torch.zeros(2, 5, dtype=torch.int32, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta")
    pages = _meta(9, 2, 16, 64)
    out = paged_attention(_meta(2, 4, 1, 64, requires_grad=True), pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        out.sum().backward()
    with pytest.raises(RuntimeError, match="records no gradient"):
        paged_append(_meta(2, 2, 1, 64, requires_grad=True), _meta(2, 2, 1, 64), pages, pages, table, lens)
    with torch.no_grad():
        assert paged_append(_meta(2, 2, 1, 64, requires_grad=True), _meta(2, 2, 1, 64), pages, pages, table, lens) is None


def test_convertible_and_other_arguments():
    q, k = _meta(2, 4, 5, 64), _meta(2, 2, 7, 64)
    assert cross_attention(q, k, k, sm_scale=1).shape == q.shape
    assert cross_attention(q, k, k, sm_scale=torch.tensor(0.5)).shape == q.shape
    with pytest.raises(RuntimeError, match="Expected a value of type"):
        cross_attention(q, k, k, sm_scale="x")


def test_references_agree_with_the_oracle():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(*s, generator=g) for s in ((2, 4, 6, 16), (2, 2, 9, 16), (2, 2, 9, 16)))
    lens, q_lens = torch.tensor([9, 0], dtype=torch.int32), torch.tensor([4, 6], dtype=torch.int32)
    out, valid = cross_attention_reference(q.double(), k.double(), v.double(), lens, q_lens)
    assert (out - kv_oracle.cross(q, k, v, lens, q_lens)["o"][0]).abs().max() < 1e-12 and valid[0].sum() == 4
    pages_k, pages_v = (torch.randn(7, 2, 4, 16, generator=g) for _ in range(2))
    table = torch.tensor([[6, 2, -1, 5], [0, 9, 1, 3]], dtype=torch.int32)
    for C, R, new in ((1, None, None), (3, 1, [2, 6]), (100, 0, None)):
        new = None if new is None else torch.tensor(new, dtype=torch.int32)
        lens = torch.tensor([15, 3], dtype=torch.int32)
        got, _ = paged_attention_reference(q.double(), pages_k.double(), pages_v.double(), table, lens, C, R, new_lens=new)
        assert (got - kv_oracle.paged(q, pages_k, pages_v, table, lens, C, R, new_lens=new)["o"][0]).abs().max() < 1e-12


def test_oracle_gradients_are_those_of_its_forward():
    g = torch.Generator().manual_seed(2)
    q, k, v, d_o = (torch.randn(*s, generator=g) for s in ((1, 4, 3, 16), (1, 2, 5, 16), (1, 2, 5, 16), (1, 4, 3, 16)))
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    lens = torch.tensor([4], dtype=torch.int32)
    out, _ = cross_attention_reference(*leaves, lens)
    want = torch.autograd.grad(out, leaves, d_o.double())
    got = kv_oracle.cross(q, k, v, lens, None, None, d_o)
    for name, w in zip(("dq", "dk", "dv"), want):
        assert (got[name][0] - w).abs().max() < 1e-12


def test_bounds_catch_a_planted_mistake():
    """One key too many, one too few, or a gradient without one head: all outside the bounds."""
    g = torch.Generator().manual_seed(3)
    q, k, v, d_o = (torch.randn(*s, generator=g).half() for s in ((1, 4, 40, 64), (1, 2, 70, 64), (1, 2, 70, 64), (1, 4, 40, 64)))
    good = kv_oracle.cross(q, k, v, torch.tensor([69]), None, None, d_o)
    for n in (70, 68):
        other = kv_oracle.cross(q, k, v, torch.tensor([n]), None, None, d_o)
        for name in ("o", "lse", "dq", "dv"):
            with pytest.raises(AssertionError):
                kv_oracle.assert_within(name, other[name][0], good[name])
    d_o[:, 3] = 0
    other = kv_oracle.cross(q, k, v, torch.tensor([69]), None, None, d_o)
    for name in ("dk", "dv"):
        with pytest.raises(AssertionError):
            kv_oracle.assert_within(name, other[name][0], good[name])
