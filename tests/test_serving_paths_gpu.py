"""Norms, rotation, pages and trees on the GPU in calls that are large enough for ways through the kernels of their own: stores past the caches,
the exchange of chunks between lanes, workgroups that find their parts by the lengths."""
import pytest
import torch

from paged_attention import paged_append_rope
from qk_norm_rope import qk_norm_rope
from tests.test_drafted_tokens_gpu import _tables
from tests.test_paged_attention_gpu import DEV, DTYPES

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
