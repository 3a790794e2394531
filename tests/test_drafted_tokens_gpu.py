"""Serving with drafted tokens on the GPU: keys turned on their way into the pages, attention of trees over them, keeping the accepted
tokens; against the float64 oracle within bounds counted in roundings, and together as a decoder uses them."""
import threading

import pytest
import torch

from oracle import kv_oracle
from paged_attention import (
    paged_append,
    paged_append_rope,
    paged_attention,
    paged_keep,
    paged_tree_attention,
    paged_tree_attention_reference,
)
from qk_norm_rope import qk_norm_rope
from tests.test_paged_attention_gpu import DEV, DTYPES, _cache, _gpu, _i32, _q
from tests.test_qk_norm_rope_gpu import _randn, _tables

pytestmark = pytest.mark.gpu


def _trees(B, T, seed=1, chain=False):
    """[B, T, T]: each token's parent is one before it, or none."""
    g = torch.Generator().manual_seed(seed)
    seen = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            parent = i - 1 if chain else int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if parent >= 0:
                seen[b, i] = seen[b, parent]
            seen[b, i, i] = True
    return seen


# ---- attention of trees ---------------------------------------------------------------------------------------------

def _check_tree(q, k, v, table, lens, tree, scale=None, new_lens=None):
    want = kv_oracle.tree(q, k, v, table, lens, tree, scale, new_lens)
    q, k, v, table, lens, tree, new_lens = _gpu(q, k, v, table, lens, tree, new_lens)
    o, lse = paged_tree_attention(q, k, v, table, lens, tree, scale, new_lens, return_lse=True)
    torch.cuda.synchronize()
    kv_oracle.assert_within("o", o, want["o"])
    kv_oracle.assert_within("lse", lse, want["lse"])
    assert torch.equal(o, paged_tree_attention(q, k, v, table, lens, tree, scale, new_lens))
    return o


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(2, 2, 1), (8, 2, 5), (3, 1, 16), (4, 4, 33), (8, 1, 9)])
@pytest.mark.parametrize("page", [1, 16, 48])
def test_trees(dtype, D, Hq, Hkv, T, page):
    lens = [T, 70 + T, 300, T + 1]
    k, v, table = _cache(lens, Hkv, D, page, dtype)
    _check_tree(_q(4, Hq, T, D, dtype), k, v, table, _i32(lens), _trees(4, T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,G,page", [(8, 4, 7), (16, 4, 64), (64, 2, 32), (70, 1, 256)])
def test_trees_over_long_caches(dtype, D, T, G, page):
    """Caches that are divided into shares, some of them empty, and joined."""
    lens = [3001, 513, T]
    k, v, table = _cache(lens, 2, D, page, dtype)
    _check_tree(_q(3, 2 * G, T, D, dtype), k, v, table, _i32(lens), _trees(1, T)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,G", [(130, 1), (100, 3), (257, 2)])
def test_large_trees(dtype, T, G):
    lens = [T + 400, T + 31, T]
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    _check_tree(_q(3, 2 * G, T, 64, dtype), k, v, table, _i32(lens), _trees(3, T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(7, 4), (40, 4), (90, 2)])
def test_any_mask(dtype, T, Hq):
    """Masks that are no tree: tokens that see none of the new ones, not even themselves, or later ones; tokens that no one sees; without a
    context rows that see nothing, and padding."""
    g = torch.Generator().manual_seed(3)
    lens = [T, T + 200, T - 3, 2, 0, T + 64]
    new = [T, T - 2, T - 3, 5, 4, 0]
    k, v, table = _cache([max(n, 1) for n in lens], 2, 64, 16, dtype)
    mask = torch.rand(6, T, T, generator=g) < 0.2
    mask[:, 1] = False
    mask[:, :, 2] = False
    _check_tree(_q(6, Hq, T, 64, dtype), k, v, table, _i32(lens), mask, new_lens=_i32(new))
    _check_tree(_q(6, Hq, T, 64, dtype), k, v, table, _i32(lens), torch.zeros(T, T, dtype=torch.bool))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(6, 4), (48, 2)])
def test_a_chain_is_causal_attention(dtype, T, Hq):
    """The same bits where the calls go the same way (up to 32 rows), the same bounds elsewhere."""
    lens = [T + 500, T, 90 + T]
    k, v, table = _cache(lens, 2, 128, 16, dtype)
    chain = torch.ones(T, T, dtype=torch.bool).tril()
    o = _check_tree(_q(3, Hq, T, 128, dtype), k, v, table, _i32(lens), chain)
    other = paged_attention(*_gpu(_q(3, Hq, T, 128, dtype), k, v, table, _i32(lens)))
    if T * Hq // 2 <= 32:
        assert torch.equal(o, other)
    want = kv_oracle.tree(_q(3, Hq, T, 128, dtype), k, v, table, _i32(lens), chain)
    kv_oracle.assert_within("o", other, want["o"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [9, 65])
def test_missing_pages_and_what_stands_in_them(dtype, T):
    """Missing pages, among them some of the drafted tokens', positions behind the length, tokens that no one sees: whatever they hold."""
    lens = [T + 150, T + 20, T]
    page = 4
    k, v, table = _cache(lens, 2, 64, page, dtype, spare=9)
    table[0, 3], table[0, (T + 140) // page], table[1, 0] = -1, 10 ** 6, -2 ** 31
    tree = _trees(3, T)
    tree[:, :, 4] = False
    q = _q(3, 4, T, 64, dtype)
    o = _check_tree(q, k, v, table, _i32(lens), tree)
    used = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            e = int(table[b, j // page])
            if 0 <= e < k.shape[0] and j != n - T + 4:
                used[e, j % page] = True
    for x in (k, v):
        x.masked_fill_(~used[:, None, :, None], float("nan"))
    assert torch.equal(paged_tree_attention(*_gpu(q, k, v, table, _i32(lens), tree)), o)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq", [(5, 8), (40, 6)])
def test_layouts_of_trees(dtype, T, Hq):
    """One tree for all, transposed and strided masks, a cache whose pages hold positions before heads, q of a packed projection."""
    lens = [T + 90, T + 300]
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    q, tree = _q(2, Hq, T, 64, dtype), _trees(1, T)[0]
    o = _check_tree(q, k, v, table, _i32(lens), tree)
    args = _gpu(q, k, v, table, _i32(lens), tree)
    wide = torch.zeros(T, 3 * T, dtype=torch.bool, device=DEV)
    wide[:, 1::3] = args[5]
    for mask in (args[5].expand(2, T, T), args[5].T.contiguous().T, wide[:, 1::3], torch.stack([args[5], ~args[5]])[:1].expand(2, T, T)):
        assert torch.equal(paged_tree_attention(*args[:5], mask), o)
    seconds = torch.stack([args[5], ~args[5]], 1)[:, 0]
    assert torch.equal(paged_tree_attention(*args[:5], seconds), o)
    swapped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in args[1:3]]
    packed = args[0].transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.nn.functional.pad(args[0], (1, 2))[..., 1:-2]
    for query in (packed, odd):
        assert torch.equal(paged_tree_attention(query, *swapped, *args[3:]), o)
    table2 = torch.nn.functional.pad(args[3], (0, 5), value=-1)[:, :args[3].shape[1]]
    pairs = torch.stack([args[4], args[4]], 1)[:, 0]
    assert torch.equal(paged_tree_attention(*args[:3], table2, pairs, args[5]), o)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_and_references(dtype):
    lens, T = [150, 40], 12
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    q, tree = _q(2, 4, T, 64, dtype), _trees(2, T)
    for scale in (0.0, -0.3, 1.0):
        _check_tree(q, k, v, table, _i32(lens), tree, scale)
    got, valid = paged_tree_attention_reference(*[t.double() for t in (q, k, v)], table, _i32(lens), tree, new_lens=_i32([12, 3]))
    want = kv_oracle.tree(q, k, v, table, _i32(lens), tree, None, _i32([12, 3]))["o"][0]
    assert (got - want).abs().max() < 1e-12 and valid.sum() == 15


def test_sequences_do_not_change_each_other():
    """The bits of a sequence are those of the same call with other lengths and values beside it."""
    T, page = 20, 16
    for Hq in (2, 8):
        k, v, table = _gpu(*_cache([900, 900, 900], 2, 128, page, torch.bfloat16))
        q, tree = _q(3, Hq, T, 128, torch.bfloat16).to(DEV), _trees(3, T).to(DEV)
        a = paged_tree_attention(q, k, v, table, _i32([900, 333, 20]).to(DEV), tree)
        q[::2] *= 2
        b = paged_tree_attention(q, k, v, table, _i32([21, 333, 900]).to(DEV), tree)
        assert torch.equal(a[1], b[1])


# ---- into the pages -------------------------------------------------------------------------------------------------

def _rope_rows(x, live, at, tables, w, eps, interleaved):
    """(value, bound) of turned rows [B, H, T, D]; zeros where a token is not live."""
    mask = live[:, None].expand(x.shape[:3])
    angles = [t[at.clamp(0, t.shape[0] - 1)][:, None].expand(*x.shape[:3], -1)[mask] for t in tables]
    full = [torch.zeros(x.shape, dtype=torch.float64) for _ in range(2)]
    for part, value in zip(full, kv_oracle.rope_rows(x[mask], *angles, w, eps, interleaved)):
        part[mask] = value
    return tuple(full)


def _check_append(q, k, v, k_pages, v_pages, table, lens, tables, w=(None, None), new_lens=None, positions=None, eps=None, interleaved=False):
    B, _, T, _ = q.shape
    N, _, page, _ = k_pages.shape
    count = torch.full((B,), T) if new_lens is None else new_lens.long().clamp(0, T)
    i = torch.arange(T)
    place = lens.long()[:, None] - count[:, None] + i
    at = place if positions is None else positions.long()
    live = (i < count[:, None]) & (at >= 0) & (at < tables[0].shape[0])
    want_q, want_k = (_rope_rows(x, live, at, tables, wx, eps, interleaved) for x, wx in zip((q, k), w))
    entry = table.long().gather(1, place.div(page, rounding_mode="floor").clamp(0, table.shape[1] - 1))
    put = live & (place >= 0) & (place < table.shape[1] * page) & (entry >= 0) & (entry < N)
    keys, bound, values = k_pages.double(), torch.zeros(k_pages.shape, dtype=torch.float64), v_pages.clone()
    for b, t in torch.nonzero(put).tolist():
        e, slot = int(entry[b, t]), int(place[b, t]) % page
        keys[e, :, slot], bound[e, :, slot], values[e, :, slot] = want_k[0][b, :, t], want_k[1][b, :, t], v[b, :, t]
    kp, vp = k_pages.to(DEV), v_pages.to(DEV)
    got = paged_append_rope(*_gpu(q, k, v), kp, vp, *_gpu(table, lens), *_gpu(*tables), *_gpu(*w), *_gpu(new_lens, positions), eps, interleaved)
    torch.cuda.synchronize()
    kv_oracle.assert_within("q", got, want_q)
    kv_oracle.assert_within("keys", kp, (keys, bound), finite=False)
    assert torch.equal(vp.cpu(), values)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T,page", [(1, 16), (9, 1), (40, 7), (3, 100)])
@pytest.mark.parametrize("norm,interleaved", [(True, False), (False, True)])
def test_append_rope(dtype, D, T, page, norm, interleaved):
    g = torch.Generator().manual_seed(T)
    lens = [T, 2 * T + 33, 100 + T]
    k_pages, v_pages, table = _cache(lens, 2, D, page, dtype)
    q, k, v = (_randn(g, dtype, 3, h, T, D) for h in (6, 2, 2))
    w = [(1 + 0.3 * _randn(g, torch.float32, D)).to(dtype) for _ in range(2)] if norm else (None, None)
    _check_append(q, k, v, k_pages, v_pages, table, _i32(lens), _tables(200, max(16, D // 2)), w, eps=1e-6 if norm else None, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_rope_leaves_out_what_has_no_place(dtype):
    """New tokens that are fewer, before the beginning, past the table, on missing pages, at positions without angles."""
    g = torch.Generator().manual_seed(4)
    T, D, page = 10, 64, 8
    lens, new = [10, 40, 4, 70, 33, 0], [10, 3, 10, 10, 0, 5]
    k_pages, v_pages, table = _cache([40] * 6, 3, D, page, dtype)
    table[1, 4] = -1
    table[0, 0] = k_pages.shape[0]
    q, k, v = (_randn(g, dtype, 6, h, T, D) for h in (3, 3, 3))
    _check_append(q, k, v, k_pages, v_pages, table, _i32(lens), _tables(100, D), new_lens=_i32(new))
    _check_append(q, k, v, k_pages, v_pages, table, _i32(lens), _tables(37, D), new_lens=_i32(new))
    at = torch.randint(-3, 45, (6, T), generator=g, dtype=torch.int32)
    _check_append(q, k, v, k_pages, v_pages, table, _i32(lens), _tables(37, D), new_lens=_i32(new), positions=at, eps=None)
    _check_append(q, k, v, k_pages, v_pages, table, _i32([2 ** 31 - 1, -2 ** 31, 40, 40, 40, 40]), _tables(50, D), positions=at)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [False, True])
def test_append_rope_is_rope_and_append(dtype, packed):
    """The same bits as one after the other, for any layout of the projection and of the cache."""
    g = torch.Generator().manual_seed(5)
    B, Hq, Hkv, T, D, page = 4, 12, 4, 70, 128, 16
    lens = _i32([70, 200, 133, 71]).to(DEV)
    k_pages, v_pages, table = _gpu(*_cache([200] * B, Hkv, D, page, dtype))
    if packed:
        qkv = _randn(g, dtype, B, T, Hq + 2 * Hkv, D).to(DEV).transpose(1, 2)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        k_pages, v_pages = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k_pages, v_pages))
    else:
        q, k, v = (_randn(g, dtype, B, h, T, D).to(DEV) for h in (Hq, Hkv, Hkv))
    w = [(1 + 0.3 * _randn(g, torch.float32, D)).to(dtype).to(DEV) for _ in range(2)]
    tables = [t.to(DEV) for t in _tables(200, 96)]
    other = [x.clone() for x in (k_pages, v_pages)]
    positions = (lens[:, None] - T + torch.arange(T, device=DEV)).int()
    turned = qk_norm_rope(q, k, *tables, *w, positions=positions)
    paged_append(turned[1], v, *other, table, lens)
    got = paged_append_rope(q, k, v, k_pages, v_pages, table, lens, *tables, *w, eps=1e-6)
    assert torch.equal(got, turned[0]) and torch.equal(k_pages, other[0]) and torch.equal(v_pages, other[1])


def test_append_rope_without_a_cache():
    """No page, or no entry in the table: the queries are turned all the same."""
    q, k = torch.randn(2, 4, 3, 64, device=DEV), torch.randn(2, 2, 3, 64, device=DEV)
    tables = [t.to(DEV) for t in _tables(9, 64)]
    lens = _i32([3, 9]).to(DEV)
    positions = (lens[:, None] - 3 + torch.arange(3, device=DEV)).int()
    want = qk_norm_rope(q, k, *tables, positions=positions, eps=None)[0]
    for pages, width in ((torch.empty(0, 2, 16, 64, device=DEV), 2), (torch.randn(4, 2, 16, 64, device=DEV), 0)):
        table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
        assert torch.equal(paged_append_rope(q, k, k, pages, pages.clone(), table, lens, *tables), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_go_as_they_are(dtype, D):
    """Every pattern of 16 bits: subnormal numbers, infinities, both zeros; what is not a number stays none."""
    v = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16).view(dtype).view(1, 1, -1, D)
    T, page = v.shape[2], 64
    q = torch.zeros(1, 1, T, D, dtype=dtype)
    pages = [torch.zeros(T // page, 1, page, D, dtype=dtype, device=DEV) for _ in range(2)]
    table = torch.arange(T // page, dtype=torch.int32)[None]
    paged_append_rope(*_gpu(q, q, v), *pages, *_gpu(table, _i32([T]), *_tables(T, 16)), eps=1e-6)
    got, want = pages[1].cpu().flatten(), v.flatten()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan) and torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan])


# ---- accepted tokens ------------------------------------------------------------------------------------------------

def _keep_by_hand(k, v, table, first, kept):
    N, _, page, _ = k.shape
    for b, path in enumerate(kept.tolist()):
        before = -1
        for i, j in enumerate(path):
            if j <= before:
                break
            before = j
            places = []
            for at in (int(first[b]) + j, int(first[b]) + i):
                e = int(table[b, at // page]) if 0 <= at < table.shape[1] * page else -1
                places.append((e, at % page) if 0 <= e < N else None)
            if None not in places:
                (e0, s0), (e1, s1) = places
                for x in (k, v):
                    x[e1, :, s1] = x[e0, :, s0].clone()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(16, 1), (64, 16), (128, 5), (256, 100)])
def test_keep(dtype, D, page):
    g = torch.Generator().manual_seed(6)
    T = 40
    first = _i32([0, 17, 100, 63, 5, 30, 1])
    k, v, table = _cache([150] * 7, 3, D, page, dtype)
    kept = torch.full((7, 23), -1, dtype=torch.int32)
    for b, n in enumerate((1, 5, 23, 0, 9)):
        kept[b, :n] = torch.randperm(T, generator=g)[:n].sort().values
    kept[5, :6] = _i32([0, 1, 2, 2, 9, 10])          # ends where it does not ascend
    kept[6, :7] = _i32([3, 4, -1, 8, 9, 10, 11])     # and at a negative entry
    want = [x.clone() for x in (k, v)]
    _keep_by_hand(*want, table, first, kept)
    for swap in (False, True):
        got = [(x.transpose(1, 2).contiguous().transpose(1, 2) if swap else x.clone()) for x in _gpu(k, v)]
        paged_keep(*got, *_gpu(table, first, kept))
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_keep_leaves_out_what_has_no_place():
    """Before the beginning, past the table, on missing pages, entries far out."""
    k, v, table = _cache([48] * 5, 2, 32, 8, torch.float32)
    table[1, 2], table[2, 1] = -1, 99
    first = _i32([-3, 14, 6, 40, 2 ** 31 - 5])
    kept = _i32([[1, 3, 5, 7, 9], [0, 2, 3, 9, 12], [2, 4, 10, 12, 13], [3, 5, 7, 8, 2 ** 31 - 1], [1, 2, 3, 9, 10]])
    want = [x.clone() for x in (k, v)]
    _keep_by_hand(*want, table, first, kept)
    got = _gpu(k, v)
    paged_keep(*got, *_gpu(table, first, kept))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("T", [5, 40])
def test_keep_of_one_cache(T):
    """Keys that are the values too move once: every entry one place, so that a second move would take the next one's."""
    k, _, table = _cache([100] * 300, 4, 128, 16, torch.bfloat16)
    first = torch.arange(300, dtype=torch.int32) % 50
    kept = torch.arange(1, T + 1, dtype=torch.int32).expand(300, T)
    want = k.clone()
    _keep_by_hand(want, want.clone(), table, first, kept)
    got = k.to(DEV)
    paged_keep(got, got, *_gpu(table, first, kept))
    assert torch.equal(got.cpu(), want)


# ---- together -------------------------------------------------------------------------------------------------------

def _decode(B, Hq, Hkv, D, page, dtype, start, depth, seed):
    """Rounds of drafting, checking and keeping beside the same tokens fed one by one; both caches and the last outputs."""
    g = torch.Generator().manual_seed(seed)
    width = 96 // page
    tables = [t.to(DEV) for t in _tables(96, D)]
    w = [(1 + 0.2 * _randn(g, torch.float32, D)).to(dtype).to(DEV) for _ in range(2)]
    shape = (B * width, Hkv, page, D)
    pages = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(4)]
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).to(DEV)
    prompt = [_randn(g, dtype, B, h, start, D).to(DEV) for h in (Hq, Hkv, Hkv)]
    lens = torch.full((B,), start, dtype=torch.int32, device=DEV)
    for cache in (pages[:2], pages[2:]):
        paged_append_rope(*prompt, *cache, table, lens, *tables, *w, eps=1e-6)
    T = 14
    for r in range(3):
        trees = _trees(B, T, seed + r)
        new = [_randn(g, dtype, B, h, T, D).to(DEV) for h in (Hq, Hkv, Hkv)]
        first = lens.clone()
        level = (trees.sum(-1) - 1).to(torch.int32).to(DEV)
        q = paged_append_rope(*new, *pages[:2], table, first + T, *tables, *w, positions=first[:, None] + level, eps=1e-6)
        out = paged_tree_attention(q, *pages[:2], table, first + T, trees.to(DEV))
        # the path to the deepest token is accepted, cut to `depth`
        kept = torch.full((B, depth), -1, dtype=torch.int32)
        for b in range(B):
            path = torch.nonzero(trees[b, trees[b].sum(-1).argmax()])[:depth, 0]
            kept[b, :len(path)] = path
        paged_keep(*pages[:2], table, first, kept.to(DEV))
        count = (kept >= 0).sum(1)
        for i in range(depth):   # one by one, in a cache of their own
            there = (kept[:, i] >= 0).to(torch.int32).to(DEV)
            pick = kept[:, i].clamp(min=0).long().to(DEV)
            one = [x[torch.arange(B, device=DEV), :, pick][:, :, None] for x in new]
            lens = lens + there
            q1 = paged_append_rope(*one, *pages[2:], table, lens, *tables, *w, new_lens=there, eps=1e-6)
            o1 = paged_attention(q1, *pages[2:], table, lens, new_lens=there)
            same = out[torch.arange(B, device=DEV), :, pick][:, :, None]
            yield there, same, o1, [lens.tolist(), table.cpu(), [p.cpu() for p in pages]] if i == depth - 1 else None
        assert lens.tolist() == (first.cpu() + count).tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 4, 64, 16), (8, 2, 128, 8)])
def test_decoding_with_drafts_gives_what_decoding_gives(dtype, Hq, Hkv, D, page):
    """Outputs of accepted tokens, and the cache afterwards: the keys to the bit, as a token's angle is that of its depth."""
    with torch.no_grad():
        for there, got, want, end in _decode(3, Hq, Hkv, D, page, dtype, 20, 4, 2):
            live = there.bool()
            # both are within the rounding of P and of the result of one value: |P| sums to 1, |v| below 5
            step = {torch.float32: 2e-5, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
            assert (got[live].float() - want[live].float()).abs().max() <= 5 * 4 * step if live.any() else True
            if end is not None:
                lens, table, pages = end
                for b, n in enumerate(lens):
                    for j in range(n):
                        e, slot = int(table[b, j // page]), j % page
                        assert torch.equal(pages[0][e, :, slot], pages[2][e, :, slot]) and torch.equal(pages[1][e, :, slot], pages[3][e, :, slot])


def _round(x):
    q = paged_append_rope(x["q"], x["k"], x["v"], x["kp"], x["vp"], x["table"], x["lens"], *x["tables"], *x["w"], positions=x["at"], eps=1e-6)
    out = paged_tree_attention(q, x["kp"], x["vp"], x["table"], x["lens"], x["tree"])
    paged_keep(x["kp"], x["vp"], x["table"], x["lens"] - x["q"].shape[2], x["kept"])
    return out


def _state(dtype, B, Hq, Hkv, T, D, L, seed):
    g = torch.Generator().manual_seed(seed)
    lens = [L - 7 * b for b in range(B)]
    kp, vp, table = _cache(lens, Hkv, D, 16, dtype, seed=seed)
    trees = _trees(B, T, seed)
    first = torch.tensor(lens) - T
    x = dict(q=_randn(g, dtype, B, Hq, T, D), k=_randn(g, dtype, B, Hkv, T, D), v=_randn(g, dtype, B, Hkv, T, D), kp=kp, vp=vp, table=table,
             lens=_i32(lens), at=(first[:, None] + trees.sum(-1) - 1).to(torch.int32), tree=trees, kept=_i32([[0, T // 2, T - 1]] * B))
    x = {n: t.to(DEV) for n, t in x.items()}
    x["tables"] = [t.to(DEV) for t in _tables(L, D)]
    x["w"] = [(1 + 0.2 * _randn(g, torch.float32, D)).to(dtype).to(DEV) for _ in range(2)]
    return x


ROUNDS = [(torch.float32, 2, 4, 2, 5, 64, 200), (torch.float16, 4, 8, 8, 12, 64, 2500), (torch.bfloat16, 16, 32, 8, 16, 128, 3000),
          (torch.bfloat16, 3, 16, 2, 64, 128, 1500)]


@pytest.mark.parametrize("shape", ROUNDS)
def test_two_graphs_of_a_round(shape):
    """A round of drafted decoding captured twice, replayed in turn and on two streams at once, with eager rounds between."""
    with torch.no_grad():
        _round(_state(*shape, 9))
        torch.cuda.synchronize()
        static, graphs, outs = [_state(*shape, s) for s in (1, 2)], [], []
        for x in static:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(_round(x))
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in graphs]
        for seeds in ((1, 2), (3, 4), (5, 6)):
            fresh = [_state(*shape, s) for s in seeds]
            for x, y in zip(static, fresh):
                for n in y:
                    for a, b in zip(x[n] if isinstance(x[n], list) else [x[n]], y[n] if isinstance(y[n], list) else [y[n]]):
                        a.copy_(b)
            for graph, stream in zip(graphs, streams):
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    graph.replay()
            torch.cuda.synchronize()
            want = [_round(y) for y in fresh]
            for x, y, out, w in zip(static, fresh, outs, want):
                assert torch.equal(out, w) and torch.equal(x["kp"], y["kp"]) and torch.equal(x["vp"], y["vp"])


def test_host_threads():
    """Rounds from several threads, each on a stream of its own."""
    with torch.no_grad():
        want = []
        for i, s in enumerate(ROUNDS):
            x = _state(*s, i)
            want.append((_round(x), x["kp"], x["vp"]))
        torch.cuda.synchronize()
    wrong = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(stream):
            for _ in range(3):
                x = _state(*ROUNDS[i], i)
                got = (_round(x), x["kp"], x["vp"])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(ROUNDS[i])

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(ROUNDS))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_pages_past_two_to_the_31_elements():
    """Offsets in a cache beyond 32 bits: the last pages of one of 2.3e9 elements."""
    N, Hkv, page, D, T = 140000, 2, 64, 128, 12
    assert N * Hkv * page * D > 1 << 31
    kp = torch.zeros(N, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros(N, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    small = _state(torch.bfloat16, 2, 8, Hkv, T, D, 180, 5)
    own = small["kp"].shape[0]
    sixteen = small["table"].shape[1] * 16
    # the same positions in pages of 64
    table = (N - 1 - torch.arange(2 * (-(-sixteen // 64)), dtype=torch.int32)).view(2, -1).to(DEV)
    big = dict(small, kp=kp, vp=vp, table=table)
    small = dict(small, kp=small["kp"].clone(), vp=small["vp"].clone())
    for b in range(2):
        for j in range(int(small["lens"][b])):
            for x, y in ((kp, small["kp"]), (vp, small["vp"])):
                x[int(table[b, j // 64]), :, j % 64] = y[int(small["table"][b, j // 16]), :, j % 16]
    assert own < N
    with torch.no_grad():
        a, b = _round(small), _round(big)
    want = kv_oracle.HALF_STEP[torch.bfloat16]
    assert (a.float() - b.float()).abs().max() <= 4 * want * 5
    for i in range(2):
        for j in range(int(small["lens"][i])):
            assert torch.equal(kp[int(table[i, j // 64]), :, j % 64], small["kp"][int(small["table"][i, j // 16]), :, j % 16])
            assert torch.equal(vp[int(table[i, j // 64]), :, j % 64], small["vp"][int(small["table"][i, j // 16]), :, j % 16])


def test_opcheck():
    x = _state(torch.float32, 2, 4, 2, 5, 64, 60, 1)
    ops = torch.ops.alexdremov_paged_attention
    torch.library.opcheck(ops.tree_forward, (x["q"], x["kp"], x["vp"], x["table"], x["lens"], x["tree"], 0.1, None, True))
    torch.library.opcheck(ops.keep, (x["kp"], x["vp"], x["table"], x["lens"] - 5, x["kept"]))
    torch.library.opcheck(ops.append_rope, (x["q"], x["k"], x["v"], x["kp"], x["vp"], x["table"], x["lens"], *x["tables"], *x["w"], None, x["at"],
                                            1e-6, False))
