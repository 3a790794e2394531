"""The tile kernel of drafted trees, which calls with more than 32 rows of a key head and enough work take: asserted to be taken, for both numbers
of waves, for pages that hold whole copies and others, and for every layout that the rules tell apart."""
import pytest
import torch

from kv_attention import _lib
from oracle import kv_oracle
from paged_attention import paged_tree_attention
from tests.test_drafted_tokens_gpu import _check_tree, _trees
from tests.test_paged_attention_gpu import DEV, DTYPES, _cache, _gpu, _i32, _q

pytestmark = pytest.mark.gpu


def _ceil(a, b):
    return -(-a // b)


def _parts(B, Hq, Hkv, T, D, page, width, dtype):
    """(parts of a run that the tile kernel would make, parts that the call makes)"""
    rows, es = Hq // Hkv * T, 4 if dtype == torch.float32 else 2
    row_bytes, units = D * es, B * Hkv
    assert rows > 32 and (row_bytes > (512 if es == 4 else 256) or units * _ceil(rows, 32) * _ceil(page * width, 32) > (4096 if es == 4 else 8192))
    tiles, waves = _ceil(page * width, 64 if row_bytes <= 256 else 32), 2 if rows <= 64 else 4
    groups = units * _ceil(rows, waves * 32)
    places = 3 if row_bytes <= 128 else 2 if waves == 2 or row_bytes == 256 else 1
    least = 8 if groups * _ceil(tiles, 8) > 128 else 4
    most = 64 if row_bytes > 256 else 16 if waves == 4 and row_bytes <= 128 else 32
    share = max(1, min(tiles, min(most, max(least, _ceil(groups * tiles, places * 256)))))
    if es == 2 and row_bytes in (128, 256) and tiles <= 64 and groups >= places * 256:   # as many whole runs as there are places
        share = tiles
    share = max(share, _ceil(tiles, max(1, (256 << 20) // (units * rows * (D + 2) * 4))))
    bytes_ = _lib.load().kv_paged_tree_forward_workspace(B, Hq, Hkv, T, D, page, width, DTYPES.index(dtype))
    return _ceil(tiles, share), max(1, bytes_ // (units * rows * (D + 2) * 4))


def _wide(B, Hkv, rows, D, page, dtype):
    """Pages of a table that is wide enough for the tile kernel (the sequences are shorter)."""
    return _ceil(32 * (8192 // (B * Hkv * _ceil(rows, 32)) + 2), page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T,G", [(33, 1), (16, 4), (65, 1), (47, 3), (260, 1)])
@pytest.mark.parametrize("page", [16, 7])
def test_tiles(dtype, D, T, G, page):
    B, Hkv = 4, 2
    lens = [T, T + 700, T + 63, T + 1]
    width = _wide(B, Hkv, T * G, D, page, dtype)
    want, parts = _parts(B, Hkv * G, Hkv, T, D, page, width, dtype)
    assert want == parts
    k, v, table = _cache(lens, Hkv, D, page, dtype, width=width)
    _check_tree(_q(B, Hkv * G, T, D, dtype), k, v, table, _i32(lens), _trees(B, T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,G", [(12, 4), (70, 2)])
@pytest.mark.parametrize("page", [1, 32, 100, 256])
def test_tiles_of_long_caches(dtype, D, T, G, page):
    """Many parts, most of them empty for the shorter sequences; one sequence as long as the table."""
    width = _ceil(8000, page)
    lens = [page * width, 2049, 513, 64 * 8, 64 * 8 + 1, T]
    k, v, table = _cache([min(n, 8000) for n in lens], 1, D, page, dtype, width=width)
    lens[0] = min(lens[0], 8000)
    if D < 256:
        lens, table = lens + lens[1:] * 13, torch.cat([table] + [table[1:]] * 13)   # sequences that share their pages
    B = len(lens)
    if B * _ceil(T * G, 32) * _ceil(page * width, 32) > 8192 or D == 256:
        want, parts = _parts(B, G, 1, T, D, page, width, dtype)
        assert want == parts > 1
    q, trees = _q(B, G, T, D, dtype), _trees(B, T)
    some = torch.tensor([0, 1, 2, 3, 4, 5, B - 1])
    want = kv_oracle.tree(q[some], k, v, table[some], _i32(lens)[some], trees[some])
    o, lse = paged_tree_attention(*_gpu(q, k, v, table, _i32(lens), trees), return_lse=True)
    kv_oracle.assert_within("o", o[some.to(DEV)], want["o"])
    kv_oracle.assert_within("lse", lse[some.to(DEV)], want["lse"])


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("B,Hkv,T,G,D", [(64, 8, 16, 4, 128), (128, 6, 40, 1, 64), (48, 8, 50, 3, 64), (64, 4, 70, 3, 128)])
def test_as_many_sequences_as_places(dtype, B, Hkv, T, G, D):
    """Whole runs, without parts, of every length up to the table's; sequences share their pages."""
    page, span = 16, 640
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, span + 1, (B,), generator=g, dtype=torch.int32)
    lens[:5] = _i32([span, 0, T - 1, 65, 64])
    k, v, pool = _cache([span] * 4, Hkv, D, page, dtype, width=span // page)
    table = pool[torch.arange(B) % 4]
    want, parts = _parts(B, Hkv * G, Hkv, T, D, page, span // page, dtype)
    assert want == parts == 1
    q, trees = _q(B, Hkv * G, T, D, dtype), _trees(B, T)
    o, lse = paged_tree_attention(*_gpu(q, k, v, table, lens, trees), return_lse=True)
    some = torch.tensor([0, 1, 2, 3, 4, 5, 6, B - 1])
    want = kv_oracle.tree(q[some], k, v, table[some], lens[some], trees[some])
    kv_oracle.assert_within("o", o[some.to(DEV)], want["o"])
    kv_oracle.assert_within("lse", lse[some.to(DEV)], want["lse"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,G,D", [(40, 1, 64), (20, 3, 128), (90, 1, 128), (50, 3, 32), (36, 1, 256)])
@pytest.mark.parametrize("page", [16, 24])
def test_any_mask_in_tiles(dtype, T, G, D, page):
    """Rows that see nothing, tokens that no one sees, sequences shorter than their new tokens, missing pages, and NaN wherever no one looks."""
    g = torch.Generator().manual_seed(3)
    B, Hkv = 7, 2
    lens = [T, T + 200, T - 3, 2, 0, T + 64, T + 100]
    new = [T, T - 2, T - 3, 5, 4, 0, T // 2]
    width = _wide(B, Hkv, T * G, D, page, dtype)
    want, parts = _parts(B, Hkv * G, Hkv, T, D, page, width, dtype)
    assert want == parts
    k, v, table = _cache([max(n, 1) for n in lens], Hkv, D, page, dtype, width=width, spare=5)
    table[1, 2], table[1, (T + 190) // page], table[6, 0], table[5, 1] = -1, k.shape[0], 2 ** 31 - 1, -2 ** 31
    mask = torch.rand(B, T, T, generator=g) < 0.2
    mask[:, 1] = False
    mask[:, :, 3] = False
    q = _q(B, Hkv * G, T, D, dtype)
    o = _check_tree(q, k, v, table, _i32(lens), mask, new_lens=_i32(new))
    used = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b, L in enumerate(lens):
        n = min(new[b], T)
        for j in range(L):
            e, u = int(table[b, j // page]), j - (L - n)
            seen = bool(mask[b, max(0, n - L):n, u].any()) if u >= 0 else n > 0
            if 0 <= e < k.shape[0] and seen:
                used[e, j % page] = True
    for x in (k, v):
        x.masked_fill_(~used[:, None, :, None], float("nan"))
    assert torch.equal(paged_tree_attention(*_gpu(q, k, v, table, _i32(lens), mask), new_lens=_i32(new).to(DEV)), o)
    assert not paged_tree_attention(*_gpu(q[:1], k[:1], v[:1], torch.full((1, width), -1, dtype=torch.int32), _i32([T]), mask[0])).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,G,D", [(16, 4, 128), (100, 1, 64)])
def test_layouts_in_tiles(dtype, T, G, D):
    """Caches whose pages hold positions before heads, keys and values of different strides, packed caches, strided masks: the same bits."""
    B, Hkv, page = 3, 2, 16
    lens = [T + 300, T, T + 77]
    width = _wide(B, Hkv, T * G, D, page, dtype)
    k, v, table = _cache(lens, Hkv, D, page, dtype, width=width)
    q, tree = _q(B, Hkv * G, T, D, dtype), _trees(1, T)[0]
    o = _check_tree(q, k, v, table, _i32(lens), tree)
    q, k, v, table, lens, tree = _gpu(q, k, v, table, _i32(lens), tree)
    swapped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    both = torch.stack([k, v], 1)
    wide = [torch.nn.functional.pad(x, (0, 32)) for x in (k, v)]
    for keys, values in (swapped, (k, swapped[1]), (swapped[0], v), (both[:, 0], both[:, 1]), [x[..., :D] for x in wide]):
        assert torch.equal(paged_tree_attention(q, keys, values, table, lens, tree), o)
    packed = q.transpose(1, 2).contiguous().transpose(1, 2)
    strided = torch.stack([tree, ~tree], 2)[..., 0]
    assert torch.equal(paged_tree_attention(packed, k, v, table, lens, strided), o)
    assert torch.equal(paged_tree_attention(packed, k, v, table, lens, strided.expand(B, T, T)), o)


def test_pages_far_apart():
    """Pages 2^31 bytes and more apart: their places do not fit the shorter way of forming them."""
    T, Hkv, page, D, width = 20, 2, 16, 64, 9000
    far = (1 << 30) + 64
    k, v, table = _cache([150], Hkv, D, page, torch.float16, width=width, spare=0)
    table[0, :10] = torch.tensor([1, 2, 0, 1, 0, 2, 2, 1, 0, 0])
    q, tree = _q(1, 4 * Hkv, T, D, torch.float16), _trees(1, T)[0]
    want = kv_oracle.tree(q, k[:3], v[:3], table, _i32([150]), tree)
    spread = []
    for x in (k, v):
        room = torch.empty(2 * far + Hkv * page * D, dtype=torch.float16, device=DEV)
        pages = room.as_strided((3, Hkv, page, D), (far, page * D, D, 1))
        pages.copy_(x[:3])
        spread.append(pages)
    o = paged_tree_attention(q.to(DEV), *spread, *_gpu(table, _i32([150]), tree))
    kv_oracle.assert_within("o", o, want["o"])


@pytest.mark.parametrize("T,G", [(16, 4), (100, 2)])
def test_sequences_do_not_change_each_other_in_tiles(T, G):
    B, Hkv, D, page = 6, 2, 128, 16
    width = _wide(B, Hkv, T * G, D, page, torch.bfloat16)
    k, v, table = _gpu(*_cache([1500] * B, Hkv, D, page, torch.bfloat16, width=width))
    q, tree = _q(B, Hkv * G, T, D, torch.bfloat16).to(DEV), _trees(B, T).to(DEV)
    a = paged_tree_attention(q, k, v, table, _i32([1500, 333, 200, 999, 1, 0]).to(DEV), tree)
    q[::2] *= 2
    q[5] *= 3
    b = paged_tree_attention(q, k, v, table, _i32([200, 333, 1500, 999, 1500, 200]).to(DEV), tree)
    assert torch.equal(a[1], b[1]) and torch.equal(a[3], b[3])
