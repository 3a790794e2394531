"""Ways through the kernels of cross attention and attention over pages that only certain sizes take, each asserted to be taken: the
hand-scheduled dK and dV beside a dQ of the tile kernel, rows by length at head dimension 256, appending past the caches, chunks of many rows."""
import pytest
import torch

from cross_attention import cross_attention
from kv_attention import _lib
from oracle import kv_oracle
from paged_attention import paged_append, paged_attention

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,lens,divided", [
    (1, 32, 8, 1000, 4224, [4100], True),                         # too few queries for a workgroup of 256 to every CU
    (1, 16, 4, 700, 8192, [8001], True),                          # likewise, in more parts
    (8, 32, 8, 300, 600, [600, 64, 0, 1, 599, 300, 128, 65], False),   # queries that fill workgroups of 256 poorly
    (5, 48, 16, 130, 520, None, False),
])
def test_dkdv_by_hand_after_dq_of_the_tile_kernel(dtype, B, Hq, Hkv, Tq, Tk, lens, divided):
    """dQ leaves the log-sum-exps and delta of grouped heads head by head, as dK and dV go through them."""
    D, G = 128, Hq // Hkv
    assert Hkv * B * -(-Tk // 128) >= 256 and G * Tq >= 384                                    # dK and dV by hand,
    assert B * Hq * -(-Tq // 256) < 256 or 4 * Tq < 3 * 256 * -(-Tq // 256)                    # dQ not
    stats = 2 * ((B * Hq * Tq * 4 + 255) // 256 * 256)
    assert (_lib.load().kv_cross_backward_workspace(B, Hq, Hkv, Tq, Tk, D, DTYPES.index(dtype)) > stats) == divided
    g = torch.Generator().manual_seed(17)
    q, k, v, d_o = (_randn(g, dtype, *s) for s in ((B, Hq, Tq, D), (B, Hkv, Tk, D), (B, Hkv, Tk, D), (B, Hq, Tq, D)))
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o, lse = cross_attention(*leaves, None if lens is None else lens.to(DEV), return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, leaves, d_o.to(DEV))
    torch.cuda.synchronize()
    for b in range(B):
        for h in sorted({0, Hkv - 1, b % Hkv}):
            heads = slice(h * G, (h + 1) * G)
            one = [t[b:b + 1] for t in (q[:, heads], k[:, h:h + 1], v[:, h:h + 1], d_o[:, heads])]
            want = kv_oracle.cross(*one[:3], None if lens is None else lens[b:b + 1], None, None, one[3])
            for name, got in (("o", o[b:b + 1, heads]), ("lse", lse[b:b + 1, heads]), ("dq", dq[b:b + 1, heads]),
                              ("dk", dk[b:b + 1, h:h + 1]), ("dv", dv[b:b + 1, h:h + 1])):
                kv_oracle.assert_within(f"{name} of {b}, key head {h}", got, want[name])


def _parts(bytes_, pairs, rows, D):
    """Parts of a run of keys, from the workspace that a call asks for."""
    return bytes_ // (pairs * rows * (D + 2) * 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_of_many_lengths_at_head_dimension_256(dtype):
    B, Hq, Hkv, Tk, D = 72, 8, 4, 2200, 256
    bytes_ = _lib.load().kv_cross_forward_workspace(B, Hq, Hkv, 1, Tk, D, DTYPES.index(dtype))
    parts = _parts(bytes_, B * Hkv, Hq // Hkv, D)
    assert parts > 1 and B * Hkv * parts >= 512
    g = torch.Generator(device=DEV).manual_seed(5)
    lens = torch.randint(0, Tk + 1, (B,), generator=g, device=DEV).to(torch.int32)
    lens[0], lens[1], lens[63], lens[64], lens[-1] = 0, Tk, 1, 1025, 0
    q, k, v = (_randn(g, dtype, *s) for s in ((B, Hq, 1, D), (B, Hkv, Tk, D), (B, Hkv, Tk, D)))
    o, lse = cross_attention(q, k, v, lens, return_lse=True)
    some = [0, 1, 2, 62, 63, 64, 65, B - 1]
    want = kv_oracle.cross(q[some].cpu(), k[some].cpu(), v[some].cpu(), lens[some].cpu())
    kv_oracle.assert_within("o", o[some], want["o"])
    kv_oracle.assert_within("lse", lse[some], want["lse"])
    order = torch.randperm(B, generator=g, device=DEV)
    assert torch.equal(cross_attention(q[order], k[order], v[order], lens[order]), o[order])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,R", [(70, 1, 1, None), (129, 2, 1, 2500), (66, 3, 64, 40)])
def test_pages_of_many_lengths_at_head_dimension_256(dtype, B, T, C, R):
    Hkv, D, page, longest = 4, 256, 16, 3100
    width = -(-longest // page)
    bytes_ = _lib.load().kv_paged_forward_workspace(B, 2 * Hkv, Hkv, T, D, page, width, C, 2 ** 31 - 1 if R is None else R, DTYPES.index(dtype))
    parts = _parts(bytes_, B * Hkv, 2 * T, D)
    assert parts > 1 and B * Hkv * parts >= 512
    g = torch.Generator(device=DEV).manual_seed(B + T)
    lens = torch.randint(0, 400, (B,), generator=g, device=DEV).to(torch.int32)
    lens[5], lens[6], lens[7], lens[20] = longest, 1, 513, 2048
    lens[0], lens[-1], lens[63], lens[64] = 0, 3000, 2500, 700
    new = None if T == 1 else torch.randint(0, T + 1, (B,), generator=g, device=DEV).to(torch.int32)
    pages = 1000
    table = torch.randint(0, pages, (B, width), generator=g, device=DEV).to(torch.int32)   # shared pages; some are not there
    table[torch.rand(B, width, generator=g, device=DEV) < 0.05] = -1
    q = _randn(g, dtype, B, 2 * Hkv, T, D)
    k, v = (_randn(g, dtype, pages, Hkv, page, D) for _ in range(2))
    o, lse = paged_attention(q, k, v, table, lens, C, R, None, new, return_lse=True)
    some = [0, 5, 6, 7, 20, 62, 63, 64, B - 1]
    want = kv_oracle.paged(q[some].cpu(), k.cpu(), v.cpu(), table[some].cpu(), lens[some].cpu(), C, R, None, None if new is None else new[some].cpu())
    kv_oracle.assert_within("o", o[some], want["o"])
    kv_oracle.assert_within("lse", lse[some], want["lse"])
    order = torch.randperm(B, generator=g, device=DEV)
    again = paged_attention(q[order], k, v, table[order], lens[order], C, R, None, None if new is None else new[order])
    assert torch.equal(again, o[order])


@pytest.mark.parametrize("dtype,B,H,T,D", [(torch.bfloat16, 8, 8, 2048, 128), (torch.float32, 5, 3, 2500, 128), (torch.float16, 7, 5, 2100, 256)])
def test_prompts_into_the_cache(dtype, B, H, T, D):
    """More bytes than the caches of the GPU hold at once: every token where it belongs, nothing else touched, and attention right after it."""
    page = 48
    assert B * H * T * D * dtype.itemsize * 2 > 32 << 20
    g = torch.Generator(device=DEV).manual_seed(12)
    new = torch.randint(0, T + 1, (B,), generator=g, device=DEV).to(torch.int32)
    new[0], new[1], new[2] = T, 0, 1
    before = torch.randint(0, 300, (B,), generator=g, device=DEV).to(torch.int32)
    before[0], before[3] = 0, -40                                          # the first tokens of sequence 3 are below position 0
    lens = before + new
    width = -(-(T + 100) // page)                                          # some of the last tokens are past the table
    pages = B * width + 5
    table = torch.randperm(pages, generator=g, device=DEV)[:B * width].view(B, width).to(torch.int32)
    table[0, 2], table[2, 0], table[4, 7] = -1, pages + 3, pages
    k, v = (_randn(g, dtype, B, H, T, D) for _ in range(2))
    k_pages, v_pages = (_randn(g, dtype, pages, H, page, D) for _ in range(2))
    want_k, want_v = k_pages.clone(), v_pages.clone()
    i = torch.arange(T, device=DEV)
    at = (before[:, None] + i).long()
    to = table.long().gather(1, (at // page).clamp(0, width - 1))
    b, t = torch.nonzero((i < new[:, None]) & (at >= 0) & (at < width * page) & (to >= 0) & (to < pages), as_tuple=True)
    want_k[to[b, t], :, at[b, t] % page], want_v[to[b, t], :, at[b, t] % page] = k[b, :, t], v[b, :, t]
    q = _randn(g, dtype, B, 2 * H, 1, D)
    with torch.no_grad():
        paged_append(k, v, k_pages, v_pages, table, lens, new)
        o = paged_attention(q, k_pages, v_pages, table, lens)
        assert torch.equal(o, paged_attention(q, want_k, want_v, table, lens))
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,T,lens,new_lens,C,R", [
    (4, 2, 64, 300, [1300, 300, 77, 0], [300, 299, 77, 5], 1, None),      # a prefix, a prompt, a short one, tokens below position 0
    (3, 1, 128, 300, [901, 640, 300, 512], [300, 33, 0, 256], 1, 100),     # windows
    (2, 2, 32, 1000, [1500, 1000], [1000, 471], 64, 3),                    # chunks
])
def test_many_new_tokens(dtype, Hq, Hkv, D, T, lens, new_lens, C, R):
    """Prompts, and further turns over what the cache holds, with pages that are not there."""
    B, page = len(lens), 16
    width = -(-max(lens) // page) + 1
    g = torch.Generator().manual_seed(14)
    pages = B * width
    table = torch.randperm(pages, generator=g).view(B, width).to(torch.int32)
    table[0, 3], table[1, 1] = -1, pages
    q = _randn(g, dtype, B, Hq, T, D)
    k, v = (_randn(g, dtype, pages, Hkv, page, D) for _ in range(2))
    lens, new = (torch.tensor(x, dtype=torch.int32) for x in (lens, new_lens))
    want = kv_oracle.paged(q, k, v, table, lens, C, R, None, new)
    o, lse = paged_attention(*(x.to(DEV) for x in (q, k, v, table, lens)), C, R, None, new.to(DEV), return_lse=True)
    kv_oracle.assert_within("o", o, want["o"])
    kv_oracle.assert_within("lse", lse, want["lse"])
