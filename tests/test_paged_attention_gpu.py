"""Attention over a cache in pages, and appending to it, on the GPU: against the float64 oracle within bounds counted in
roundings, and against the streaming attention whose last rows it gives."""
import pytest
import torch

from oracle import kv_oracle
from paged_attention import paged_append, paged_attention, paged_attention_reference
from streaming_attention import streaming_attention

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _cache(lens, Hkv, D, page, dtype, seed=5, width=None, spare=3, fill=None):
    """(k_pages, v_pages, table): every sequence has its pages anywhere in the cache; -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    width = max(need + [1]) if width is None else width
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn(total, Hkv, page, D, generator=g).to(dtype) for _ in range(2))
    if fill is not None:
        k[:], v[:] = fill, fill
    return k, v, table


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def _gpu(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _check(q, k, v, table, lens, C=1, R=None, scale=None, new_lens=None):
    want = kv_oracle.paged(q, k, v, table, lens, C, R, scale, new_lens)
    q, k, v, table, lens, new_lens = _gpu(q, k, v, table, lens, new_lens)
    o, lse = paged_attention(q, k, v, table, lens, C, R, scale, new_lens, return_lse=True)
    torch.cuda.synchronize()
    kv_oracle.assert_within("o", o, want["o"])
    kv_oracle.assert_within("lse", lse, want["lse"])
    assert torch.equal(o, paged_attention(q, k, v, table, lens, C, R, scale, new_lens))
    return o


def _q(B, Hq, T, D, dtype, seed=6):
    return torch.randn(B, Hq, T, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (3, 1), (40, 1)])
@pytest.mark.parametrize("page", [1, 16, 48])
def test_one_token(dtype, D, Hq, Hkv, page):
    lens = [1, 33, 700, 0]
    k, v, table = _cache(lens, Hkv, D, page, dtype)
    _check(_q(4, Hq, 1, D, dtype), k, v, table, _i32(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [7, 32, 256])
def test_long_caches(dtype, D, page):
    """Caches that are divided into shares, some of them empty, and joined."""
    lens = [5000, 513, 2]
    k, v, table = _cache(lens, 2, D, page, dtype)
    _check(_q(3, 4, 1, D, dtype), k, v, table, _i32(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,R", [(1, None), (1, 0), (1, 40), (8, 2), (32, 0), (10, 9), (1000, 0), (13, None)])
@pytest.mark.parametrize("T,new_lens", [(1, None), (5, [5, 3, 0, 1]), (40, [40, 12, 40, 33])])
def test_windows(dtype, C, R, T, new_lens):
    lens = [100, 45, 40, 640]
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    _check(_q(4, 6, T, 64, dtype), k, v, table, _i32(lens), C, R, new_lens=_i32(new_lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,R,T", [(16, 3, 16), (10, 9, 10), (1, 50, 4)])
def test_same_as_the_last_rows_of_streaming_attention(dtype, C, R, T):
    """Tokens appended in pieces; their attention is that of the rows of the whole sequence."""
    B, H, D, page, total = 3, 4, 64, 16, 173
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(B, H, total, D, generator=g).to(dtype).to(DEV) for _ in range(3))
    k_pages, v_pages, table = _gpu(*_cache([total] * B, H, D, page, dtype, fill=float("nan")))
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    have = 0
    while have < total:
        n = min(T, total - have)
        lens += n
        new = torch.full((B,), n, dtype=torch.int32, device=DEV)
        piece = slice(have, have + T)
        chunk = [torch.nn.functional.pad(x[:, :, piece], (0, 0, 0, T - n)) for x in (q, k, v)]
        with torch.no_grad():
            paged_append(chunk[1], chunk[2], k_pages, v_pages, table, lens, new)
            got = paged_attention(chunk[0], k_pages, v_pages, table, lens, C, R, new_lens=new)
        have += n
        whole = streaming_attention(*(x[:, :, :have].contiguous() for x in (q, k, v)), None, C, R)[:, :, have - n:]
        # both within the rounding of P and of the result: |P| sums to 1, |v| below 5
        step = {torch.float32: 2e-5, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
        assert (got[:, :, :n].float() - whole.float()).abs().max() <= 5 * 4 * step
        assert not got[:, :, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
@pytest.mark.parametrize("C,R", [(1, None), (1, 30)])
def test_what_no_token_sees_does_not_matter(dtype, D, junk, C, R):
    lens, page = [50, 131, 7], 12
    k, v, table = _cache(lens, 2, D, page, dtype, width=20)
    q = _q(3, 4, 1, D, dtype)
    clean = paged_attention(*_gpu(q, k, v, table, _i32(lens)), C, R)
    kj, vj = torch.full_like(k, junk), torch.full_like(v, junk)
    for b, n in enumerate(lens):
        first = 0 if R is None else max(0, n - 1 - R)
        for t in range(first, n):
            e = int(table[b, t // page])
            kj[e, :, t % page], vj[e, :, t % page] = k[e, :, t % page], v[e, :, t % page]
    dirty = paged_attention(*_gpu(q, kj, vj, table, _i32(lens)), C, R)
    assert torch.isfinite(dirty).all() and torch.equal(clean, dirty)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, 23])
def test_pages_that_are_not_there(dtype, bad):
    """Their positions are not seen, in the middle of a sequence or all of it."""
    lens = [90, 50, 33, 600]
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    bad = len(k) if bad == 23 else bad
    table[0, 2] = bad
    table[1, :] = bad
    table[2, 0], table[2, 2] = bad, bad
    table[3, 5:30] = bad
    for T in (1, 3):
        o = _check(_q(4, 4, T, 64, dtype), k, v, table, _i32(lens))
        assert not o[1].any()


def test_no_pages_at_all():
    q, lens = _q(2, 4, 2, 64, torch.float16).to(DEV), torch.tensor([5, 0], dtype=torch.int32, device=DEV)
    none = torch.zeros(0, 2, 16, 64, dtype=torch.float16, device=DEV)
    some = torch.ones(3, 2, 16, 64, dtype=torch.float16, device=DEV)
    for pages, width in ((none, 4), (some, 0), (none, 0)):
        table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
        o, lse = paged_attention(q, pages, pages, table, lens, return_lse=True)
        assert not o.any() and (lse == -float("inf")).all()
        with torch.no_grad():
            paged_append(q[:, :2].contiguous(), q[:, :2].contiguous(), pages, pages.clone(), table, lens)
    assert (some == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lengths_beyond_the_table_and_below_zero(dtype):
    lens = [48, 48, 48]
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    q = _q(3, 2, 1, 64, dtype)
    want = _check(q, k, v, table, _i32([48, 48, 0]))
    got = paged_attention(*_gpu(q, k, v, table, _i32([1000, 2 ** 31 - 1, -5])))
    assert torch.equal(got, want) and not got[2].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Caches stored as [pages, page_size, heads, head_dim], both in one tensor, a table cut from a larger one."""
    lens, page = [70, 20], 16
    k, v, table = _cache(lens, 2, 64, page, dtype)
    q = _q(2, 4, 3, 64, dtype)
    want = paged_attention(*_gpu(q, k, v, table, _i32(lens)))
    joint = torch.stack([k, v], 1).to(DEV)
    other = [x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (k, v)]
    large = torch.full((4, table.shape[1] + 5), 7, dtype=torch.int32)
    large[::2, 2:2 + table.shape[1]] = table
    cut = large.to(DEV)[::2, 2:2 + table.shape[1]]
    q_t = q.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    l2 = torch.tensor([[70, 1], [20, 1]], dtype=torch.int32, device=DEV)[:, 0]
    for kk, vv in ((joint[:, 0], joint[:, 1]), other):
        assert torch.equal(paged_attention(q_t, kk, vv, cut, l2), want)
    assert torch.equal(paged_attention(q_t, *other, cut.t().contiguous().t(), l2), want)
    ref, _ = paged_attention_reference(*_gpu(q.float(), k.float(), v.float(), table, _i32(lens)))
    assert (want.float() - ref).abs().max() < (1e-4 if dtype == torch.float32 else 4 * 5 * 2.0 ** -8)


def test_long_cache_offsets():
    """Pages whose places in the cache pass 32 bits of bytes and of elements."""
    D, page = 64, 64
    pages = (9 << 30) // (page * D * 2)   # 9 GiB
    big = torch.empty(pages, 1, page, D, dtype=torch.float16, device=DEV)
    k, v, table = _cache([300], 1, D, page, torch.float16)
    at = torch.tensor([pages - 1, 3, pages // 2 + 1, pages - 7, pages // 4 * 3], dtype=torch.int32)
    for i, e in enumerate(at.tolist()):
        big[e] = k[int(table[0, i])].to(DEV)
    q = _q(1, 2, 1, D, torch.float16)
    want = paged_attention(*_gpu(q, k, k, table, _i32([300])))
    assert torch.equal(paged_attention(q.to(DEV), big, big, at[None].to(DEV), _i32([300]).to(DEV)), want)
    new = torch.ones(1, 1, 1, D, dtype=torch.float16, device=DEV)
    paged_append(new, new, big, big, at[None].to(DEV), _i32([20]).to(DEV))
    assert (big[pages - 1, 0, 19] == 1).all() and torch.equal(big[pages - 1, 0, 20].cpu(), k[int(table[0, 0]), 0, 20])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [5, 150])
def test_same_bits_whatever_the_other_sequences(dtype, B):
    lens = [900, 2000, 17, 1300, 64] + [40] * (B - 5)
    k, v, table = _cache(lens, 2, 64, 16, dtype)
    q, k, v, table, lens = _gpu(_q(B, 8, 2, 64, dtype), k, v, table, _i32(lens))
    whole = paged_attention(q, k, v, table, lens)
    assert torch.equal(paged_attention(q, k, v, table, lens), whole)
    for b in range(5):
        others = torch.where(torch.arange(B, device=DEV) == b, lens, lens // 3)
        moved = q.roll(1, 0)
        moved[b] = q[b]
        assert torch.equal(paged_attention(moved, k, v, table, others)[b], whole[b])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("B,T", [(1, 3000), (40, 1500), (300, 700), (300, 100)])
def test_every_division_of_the_work(dtype, D, B, T):
    """Few and many workgroups, short and long shares: every number of waves."""
    lens = [T - 37 * (b % 7) for b in range(B)]
    g = torch.Generator().manual_seed(3)
    pages = (T + 15) // 16
    k, v = (torch.randn(pages, 2, 16, D, generator=g).to(dtype) for _ in range(2))
    table = torch.stack([torch.arange(pages).roll(b) for b in range(B)]).to(torch.int32)   # all share the pages
    q = _q(B, 4, 1, D, dtype)
    got = paged_attention(*_gpu(q, k, v, table, _i32(lens)))
    some = sorted({0, B // 2, B - 1})
    want = kv_oracle.paged(q[some], k, v, table[some], _i32([lens[b] for b in some]))
    kv_oracle.assert_within("o", got[some], want["o"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,T,C,R", [(70, 1, 1, None), (200, 1, 1, None), (129, 2, 1, 2500), (66, 3, 64, 40), (256, 1, 1, None)])
def test_parts_by_length(dtype, D, B, T, C, R):
    """Batches of every length, whose parts the workgroups find from the lengths: some sequences against the oracle, and all against
    the same call with the sequences in another order."""
    Hkv, longest = 4, 3100
    g = torch.Generator().manual_seed(B + T)
    lens = torch.randint(0, 400, (B,), generator=g)
    lens[torch.randperm(B, generator=g)[:9]] = torch.tensor([longest, 0, 1, 2999, 512, 513, 1024, 2048, 1600])
    lens[0], lens[-1], lens[63], lens[64] = 0, 3000, 2500, 700
    new_lens = None if T == 1 else torch.randint(0, T + 1, (B,), generator=g).to(torch.int32)
    q = _q(B, 2 * Hkv, T, D, dtype)
    k, v, table = _cache(lens.tolist(), Hkv, D, 16, dtype)
    lens = lens.to(torch.int32)
    on = _gpu(q, k, v, table, lens)
    new = None if new_lens is None else new_lens.to(DEV)
    o, lse = paged_attention(*on, C, R, None, new, return_lse=True)
    some = [0, 1, 2, 62, 63, 64, B - 2, B - 1, int(lens.argmax())]
    want = kv_oracle.paged(q[some], k, v, table[some], lens[some], C, R, None, None if new_lens is None else new_lens[some])
    kv_oracle.assert_within("o", o[some], want["o"])
    kv_oracle.assert_within("lse", lse[some], want["lse"])
    order = torch.randperm(B, generator=g).to(DEV)
    again, _ = paged_attention(on[0][order], on[1], on[2], on[3][order], on[4][order], C, R, None, None if new is None else new[order], return_lse=True)
    assert torch.equal(again, o[order])
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 64, 256])
@pytest.mark.parametrize("T,page,lens,new_lens", [(1, 16, [1, 40, 16, 17], None), (5, 3, [5, 9, 40, 3], [5, 0, 2, 5]),
                                                  (70, 16, [70, 200, 71, 100], [70, 1, 64, 33]), (4, 16, [2, 100, 400, 1], None)])
def test_append(dtype, D, T, page, lens, new_lens):
    """Every new token where it belongs, and nothing else touched: positions below 0, past the table, pages not there."""
    H = 3
    k_pages, v_pages, table = _cache([min(n, 250) for n in lens], H, D, page, dtype)
    table[3, 0] = len(k_pages) + 4
    k, v = _q(4, H, T, D, dtype, 1), _q(4, H, T, D, dtype, 2)
    want_k, want_v = k_pages.clone(), v_pages.clone()
    for b in range(4):
        n = T if new_lens is None else new_lens[b]
        for i in range(n):
            at = lens[b] - n + i
            if 0 <= at < table.shape[1] * page and 0 <= int(table[b, at // page]) < len(k_pages):
                e = int(table[b, at // page])
                want_k[e, :, at % page], want_v[e, :, at % page] = k[b, :, i], v[b, :, i]
    got_k, got_v = _gpu(k_pages, v_pages)
    version = got_k._version
    paged_append(*_gpu(k, v), got_k, got_v, *_gpu(table, _i32(lens), _i32(new_lens)))
    assert torch.equal(got_k.cpu(), want_k) and torch.equal(got_v.cpu(), want_v)
    assert got_k._version > version
    # through views: a joint cache with the heads innermost, and projections read in place
    joint = torch.stack([k_pages, v_pages], 1).transpose(2, 3).contiguous().to(DEV).transpose(2, 3)
    kv = torch.stack([k, v], 2).permute(0, 3, 2, 1, 4).contiguous().to(DEV)
    paged_append(kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), joint[:, 0], joint[:, 1],
                 *_gpu(table, _i32(lens), _i32(new_lens)))
    assert torch.equal(joint[:, 0].cpu(), want_k) and torch.equal(joint[:, 1].cpu(), want_v)


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_decoding_with_graph(dtype):
    """Steps of append and attention captured once and replayed; lengths advance on the GPU."""
    B, Hq, Hkv, D, page, steps = 3, 8, 2, 64, 16, 6
    g = torch.Generator().manual_seed(21)
    start = [10, 515, 31]
    q, k, v = (torch.randn(steps, B, h, 1, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hkv, Hkv))
    k0, v0, table = _gpu(*_cache([n + steps for n in start], Hkv, D, page, dtype, fill=float("nan")))
    table = torch.nn.functional.pad(table, (0, 8), value=-1)
    hist = [torch.randn(B, Hkv, max(start), D, generator=g).to(dtype).to(DEV) for _ in range(2)]

    def fresh():
        cache = k0.clone(), v0.clone()
        lens = torch.tensor(start, dtype=torch.int32, device=DEV)
        shifted = [torch.zeros_like(x) for x in hist]
        for b, n in enumerate(start):
            for s, x in zip(shifted, hist):
                s[b, :, :n] = x[b, :, :n]
        paged_append(*shifted, *cache, table, lens, lens)
        return cache, lens

    def step(x, cache, lens):
        lens += 1
        paged_append(x[1], x[2], *cache, table, lens)
        return paged_attention(x[0], *cache, table, lens)

    cache, lens = fresh()
    want = [step([t[i] for t in (q, k, v)], cache, lens).clone() for i in range(steps)]
    for w in want:
        assert torch.isfinite(w).all()
    cache, lens = fresh()
    static = [t[0].clone() for t in (q, k, v)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    kept = lens.clone()
    with torch.cuda.graph(graph):
        out = step(static, cache, lens)
    lens.copy_(kept)
    for i in range(steps):
        for s, t in zip(static, (q, k, v)):
            s.copy_(t[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        (want[i] * 2).sum().item()


def test_streams():
    lens = [3000, 1500]
    sets = [_gpu(_q(2, 8, 1, 64, torch.float16, s), *_cache(lens, 2, 64, 16, torch.float16, s), _i32(lens)) for s in (1, 2)]
    want = [paged_attention(*x) for x in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r, want[i])


def test_opcheck():
    lens = [70, 20]
    q, k, v, table, lens = _gpu(_q(2, 4, 1, 64, torch.float32), *_cache(lens, 2, 64, 16, torch.float32), _i32(lens))
    ops = torch.ops.alexdremov_paged_attention
    torch.library.opcheck(ops.forward.default, (q, k, v, table, lens, 1, 2 ** 31 - 1, 0.125, None, True))
    new = torch.randn(2, 2, 1, 64, device=DEV)
    torch.library.opcheck(ops.append.default, (new, new, k, v, table, lens, None), test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(paged_attention, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(q, k, v, table, lens), paged_attention(q, k, v, table, lens))


def test_append_and_attention_under_compile():
    lens = [70, 20]
    q, k, v, table, lens = _gpu(_q(2, 4, 1, 64, torch.float32), *_cache(lens, 2, 64, 16, torch.float32), _i32(lens))
    new = torch.randn(2, 2, 1, 64, device=DEV)

    def step(kp, vp):
        paged_append(new, new, kp, vp, table, lens)
        return paged_attention(q, kp, vp, table, lens)

    a, b = (k.clone(), v.clone()), (k.clone(), v.clone())
    with torch.no_grad():
        assert torch.equal(torch.compile(step, backend="aot_eager", fullgraph=True)(*a), step(*b))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], k)
