"""Norms, rotation, pages and trees on the GPU in calls that are large enough for ways through the kernels of their own: stores past the caches,
the exchange of chunks between lanes, workgroups that find their parts by the lengths."""
import pytest
import torch

from kv_attention import _lib
from oracle import kv_oracle
from paged_attention import paged_append_rope, paged_tree_attention
from qk_norm_rope import qk_norm_rope
from tests import test_qk_norm_rope_gpu as rope_tests
from tests.test_paged_attention_gpu import DEV, DTYPES, _cache, _gpu, _i32, _q
from tests.test_qk_norm_rope_gpu import _tables

pytestmark = pytest.mark.gpu


def _past_caches(rows, D, dtype):
    """More than the caches hold, read and written."""
    return 2 * rows * D * dtype.itemsize > 32 << 20


def _bits(x):
    return x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", [(16, 16), (64, 64), (64, 32), (128, 128), (128, 64), (256, 128)])
@pytest.mark.parametrize("T", [5, 40001])
@pytest.mark.parametrize("eps", [None, 1e-6])
def test_values_keep_every_bit(dtype, D, rot, T, eps):
    """Any bits: numbers, infinities, subnormal numbers, zeros of both signs, and what is not a number, with its sign and all that it carries."""
    g = torch.Generator(device=DEV).manual_seed(7)
    bits = torch.int16 if dtype.itemsize == 2 else torch.int32
    info = torch.iinfo(bits)
    v = torch.randint(info.min, info.max + 1, (1, 2, T, D), generator=g, device=DEV, dtype=torch.int64).to(bits).view(dtype)
    v[:, :, ::3] = torch.randint(1, 1 << (7 if dtype == torch.bfloat16 else 10), v[:, :, ::3].shape, generator=g, device=DEV).to(bits).bitwise_or(
        {torch.bfloat16: 0x7F80, torch.float16: 0x7C00, torch.float32: 0x7F800000}[dtype]).view(dtype)   # not numbers, the quiet bit not set in most
    assert T < 100 or D < 64 or _past_caches(6 * T, D, dtype)
    q = torch.zeros(1, 2, T, D, dtype=dtype, device=DEV)
    page, tables = 64, [t.to(DEV) for t in _tables(T, rot)]
    width = -(-T // page)
    pages = [torch.zeros(width, 2, page, D, dtype=dtype, device=DEV) for _ in range(2)]
    table = torch.arange(width, dtype=torch.int32, device=DEV)[None]
    paged_append_rope(q, q, v, *pages, table, torch.tensor([T], dtype=torch.int32, device=DEV), *tables, eps=eps)
    got = pages[1].transpose(0, 1).reshape(2, width * page, D)[:, :T]
    assert torch.equal(_bits(got), _bits(v[0]))


def _allocated(call):
    """(result, bytes that the call allocated at most)"""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_any_distance_apart(dtype):
    """Rows of a head further apart than 32-bit byte offsets reach: read in place, the bits of a contiguous copy."""
    Hq, Hkv, T, D = 4, 2, 600, 64
    step = (1 << 32) // dtype.itemsize // (T + 1000) // 64 * 64
    assert step * T * dtype.itemsize > 1 << 30 and step * (T + 1024) * dtype.itemsize > 1 << 32
    g = torch.Generator(device=DEV).manual_seed(1)
    far = torch.empty(step * T, dtype=dtype, device=DEV).as_strided((1, 2 * (Hq + 2 * Hkv), T, D), (0, D, step, 1))
    far.copy_(torch.randn(far.shape, generator=g, device=DEV))
    near = far.contiguous()
    tables, lens = [t.to(DEV) for t in _tables(T, D)], torch.tensor([T], dtype=torch.int32, device=DEV)
    w = torch.rand(D, generator=g, device=DEV).to(dtype)
    forward, backward = torch.ops.alexdremov_qk_norm_rope.forward, torch.ops.alexdremov_qk_norm_rope.backward
    page = 40
    table = torch.arange(T // page, dtype=torch.int32, device=DEV)[None]
    empty = torch.zeros(T // page, Hkv, page, D, dtype=dtype, device=DEV)
    results = []
    for x in (near, far):
        q, k, v, dq, dk, _ = x.split([Hq, Hkv, Hkv] * 2, dim=1)
        pages = [empty.clone(), empty.clone()]
        calls = [lambda: forward(q, k, *tables, w, w, lens, None, 1e-6, False),
                 lambda: backward(dq, dk, q, k, *tables, w, w, lens, None, 1e-6, False, False)[:2],
                 lambda: (paged_append_rope(q, k, v, *pages, table, lens, *tables, w, w, eps=1e-6),)]
        results.append([])
        for call in calls:
            out, most = _allocated(call)
            copied = x is far and most >= 1.25 * sum(t.numel() * t.element_size() for t in out)
            assert not copied, most
            results[-1] += out
        results[-1] += pages
    assert all(torch.equal(a, b) and a.any() for a, b in zip(*results))


@pytest.mark.parametrize("eps", [0.0, -1e-6, 1e-60, 3.4e38, 3.402e38, 1e39, float("inf"), float("nan")])
def test_eps_that_float32_does_not_hold(eps):
    """Refused by name, whichever way it is out of range."""
    q, table = torch.zeros(1, 1, 3, 32, device=DEV), torch.zeros(3, 16, device=DEV)
    with pytest.raises(AssertionError, match="eps must be a positive number of float32"):
        qk_norm_rope(q, q, table, table, eps=eps)
    pages, one = torch.zeros(1, 1, 4, 32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(AssertionError, match="eps must be a positive number of float32"):
        paged_append_rope(q, q, q, pages, pages.clone(), one, one[0] + 3, table, table, eps=eps)


def test_the_largest_eps():
    q = torch.ones(1, 1, 3, 32, device=DEV)
    out = qk_norm_rope(q, q, torch.ones(3, 16, device=DEV), torch.zeros(3, 16, device=DEV), eps=3.39e38)[0]
    # the root, a product: some roundings of float32
    assert ((out.double() * 3.39e38 ** 0.5 - 1).abs() <= 8 * 2.0 ** -24).all()


# ---- calls past the caches --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,D,rot,interleaved", [
    (torch.float16, 64, 64, False), (torch.bfloat16, 64, 32, False), (torch.bfloat16, 64, 32, True), (torch.float32, 32, 32, False),
    (torch.float32, 32, 16, True), (torch.float32, 64, 32, False)])
def test_large_calls_of_short_rows(dtype, D, rot, interleaved):
    """Rows of 128 bytes, of which two tokens exchange a chunk, and rows of 256 of which half is turned in float32."""
    rope_tests.test_large_calls_give_what_small_ones_give(dtype, D, rot, interleaved)


def _turned_in_pieces(q, k, tables, w, lens, at, eps, interleaved, pieces=7):
    """qk_norm_rope in calls that stay in the caches."""
    T = q.shape[2]
    out = [torch.empty(x.shape, dtype=x.dtype, device=DEV) for x in (q, k)]
    for t0 in range(0, T, -(-T // pieces)):
        t1 = min(T, t0 + -(-T // pieces))
        part = [x[:, :, t0:t1] for x in (q, k)]
        assert not _past_caches(sum(x[..., 0].numel() for x in part), q.shape[3], q.dtype)
        for to, x in zip(out, qk_norm_rope(*part, *tables, *w, lens=(lens - t0).clamp(min=0).int(), positions=at[:, t0:t1], eps=eps, interleaved=interleaved)):
            to[:, :, t0:t1] = x
    return out


@pytest.mark.parametrize("dtype,D,rot,interleaved", [
    (torch.float16, 64, 64, False), (torch.bfloat16, 64, 32, False), (torch.bfloat16, 64, 32, True), (torch.float32, 32, 32, False),
    (torch.float32, 64, 32, False), (torch.float32, 64, 64, False), (torch.bfloat16, 128, 64, False), (torch.float16, 128, 128, False),
    (torch.bfloat16, 128, 32, True), (torch.float32, 128, 64, False), (torch.bfloat16, 256, 128, False), (torch.float16, 256, 64, False)])
@pytest.mark.parametrize("page", [7, 64])
@pytest.mark.parametrize("norm,depths", [(True, False), (False, True)])
def test_large_appends(dtype, D, rot, interleaved, page, norm, depths):
    """More than the caches hold, into the pages past the caches: the bits of small calls, each where its token goes, and the rest of the cache as it
    was.  An odd number of tokens, fewer new ones for some, missing pages, tokens before the beginning, past the table and without angles."""
    B, Hq, Hkv = 3, 6, 2
    T = (20 << 20) // (B * (Hq + 2 * Hkv) * D * dtype.itemsize) | 1
    assert _past_caches(B * (Hq + 2 * Hkv) * T, D, dtype) and B * T % 2 == 1
    g = torch.Generator(device=DEV).manual_seed(8)
    qkv = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    lens = torch.tensor([T + 30, T - 5, T // 2 + 100], dtype=torch.int32, device=DEV)
    new = torch.tensor([T, T, T // 2], dtype=torch.int32, device=DEV)
    width = -(-(T + 20) // page)
    assert width * page < T + 30 or page == 64
    N = B * width + 3
    table = torch.randperm(N, generator=g, device=DEV)[:B * width].view(B, width).int()
    table[0, 3], table[1, width // 2], table[2, 5] = -1, N, -2 ** 31
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dtype) for _ in range(2)] if norm else [None, None]
    eps = 1e-6 if norm else None
    tables = [t.to(DEV) for t in _tables(T - 9, rot)]
    i = torch.arange(T, device=DEV)
    place = lens[:, None] - new[:, None] + i
    at = torch.randint(-3, T, (B, T), generator=g, device=DEV, dtype=torch.int32) if depths else place.int()
    before = [torch.randn(N, Hkv, page, D, generator=g, device=DEV).to(dtype) for _ in range(2)]
    pages = [x.clone() for x in before]
    got = paged_append_rope(q, k, v, *pages, table, lens, *tables, *w, new_lens=new, positions=at if depths else None, eps=eps, interleaved=interleaved)
    want_q, want_k = _turned_in_pieces(q, k, tables, w, new, at, eps, interleaved)
    assert torch.equal(got, want_q)
    entry = table.gather(1, (place // page).clamp(0, width - 1)).long()
    live = (i < new[:, None]) & (at >= 0) & (at < T - 9)
    put = live & (place >= 0) & (place < width * page) & (entry >= 0) & (entry < N)
    assert 0 < put.sum() < live.sum() < B * T
    to = entry[put], place[put] % page
    for have, old, x in zip(pages, before, (want_k, v)):
        old[to[0], :, to[1]] = x.transpose(1, 2)[put]
        assert torch.equal(have, old)


# ---- trees, by length ---------------------------------------------------------------------------------------------------

def _by_length(B, Hq, Hkv, T, D, page, width, dtype):
    """The rules of calls of up to 32 rows: the number of parts that the longest sequence has, where workgroups find theirs by the lengths."""
    rows, units, row_bytes, f32 = Hq // Hkv * T, B * Hkv, D * dtype.itemsize, dtype == torch.float32
    assert rows <= 32 and row_bytes >= 128 and B <= 256 and units >= 48
    tiles = -(-page * width // 32)
    share = -(-units * tiles // 256)
    assert tiles > 64 and share > 16 and units * -(-tiles // 16) >= 1024   # shares of sixteen tiles
    parts = -(-tiles // 16)
    waves = 2 if row_bytes == 512 or (row_bytes == 256 and not f32) else 1 if row_bytes == 1024 else 4
    places = 256 * (163840 // (waves * (128 * row_bytes + 1536)))
    assert units * parts >= 2 * places
    bytes_ = _lib.load().kv_paged_tree_forward_workspace(B, Hq, Hkv, T, D, page, width, DTYPES.index(dtype))
    assert bytes_ == parts * units * rows * (D + 2) * 4
    return parts


@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 32), (torch.float32, 64),
                                     (torch.float32, 128), (torch.float32, 256)])
@pytest.mark.parametrize("T,G,page", [(8, 4, 16), (5, 3, 48), (32, 1, 7)])
def test_trees_by_length(dtype, D, T, G, page):
    """A serving batch of few drafted tokens over a long table: sequences of every length, empty ones and ones that are shorter than their drafts among them,
    fewer drafts for some, masks that are no tree, missing pages, and NaN wherever no one looks."""
    B, Hkv, span = 64, 2, 8000
    width = -(-span // page)
    _by_length(B, G * Hkv, Hkv, T, D, page, width, dtype)
    g = torch.Generator().manual_seed(9)
    lens = torch.exp(torch.rand(B, generator=g) * 5 + 4).int().clamp(max=span)
    lens[:12] = _i32([span, 0, T - 1, T, 1, T + 1, 512, 513, 511 + T, 7999, 33, 4097])
    new = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    new[:12] = _i32([T, T, T, T, T, 0, T, T - 1, T, 1, T, T])
    k, v, pool = _cache([span] * 4, Hkv, D, page, dtype, width=width)
    table = pool[torch.arange(B) % 4].clone()   # (sequences that share their pages)
    table[6, 3], table[8, 0], table[11, (4097 - T // 2) // page] = -1, k.shape[0], -2 ** 31
    mask = torch.rand(B, T, T, generator=g) < 0.3
    mask[:, 1] = False
    mask[:, :, 2] = False
    q = _q(B, G * Hkv, T, D, dtype)
    some = torch.tensor([*range(12), 20, 41, B - 1])
    want = kv_oracle.tree(q[some], k, v, table[some], lens[some], mask[some], new_lens=new[some])
    o, lse = paged_tree_attention(*_gpu(q, k, v, table, lens, mask), new_lens=new.to(DEV), return_lse=True)
    torch.cuda.synchronize()
    kv_oracle.assert_within("o", o[some.to(DEV)], want["o"])
    kv_oracle.assert_within("lse", lse[some.to(DEV)], want["lse"])
    assert torch.isfinite(o).all()
    used = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b in range(B):
        L, n = int(lens[b]), int(new[b])
        seen = torch.zeros(width * page, dtype=torch.bool)
        if n > 0 and L > 0:
            seen[:max(0, L - n)] = True
            late = max(0, n - L)   # drafts before the beginning see nothing and are not seen
            seen[max(0, L - n):L] = mask[b, late:n, late:n].any(0)
        entry = table[b].long()
        there = (entry >= 0) & (entry < k.shape[0])
        used[entry[there]] |= seen.view(width, page)[there]
    for x in (k, v):
        x.masked_fill_(~used[:, None, :, None], float("nan"))
    again = paged_tree_attention(*_gpu(q, k, v, table, lens, mask), new_lens=new.to(DEV))
    assert torch.equal(again, o)
    # the bits of a sequence do not depend on the lengths and values beside it
    lens[20:40], q[20:40] = lens[20:40].flip(0), 2 * q[20:40]
    other = paged_tree_attention(*_gpu(q, k, v, table, lens, mask), new_lens=new.to(DEV))
    assert torch.equal(other[:20], o[:20]) and torch.equal(other[40:], o[40:])
