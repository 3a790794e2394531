"""Sizes at the limits of a launch, and scales at those of float32, on the host: refused by name before anything is enqueued, and one
step below them not."""
import ctypes

import pytest
import torch

from kv_attention import _lib, ops

ARG, TOO_LARGE = -3, -5
MOST_THREADS = 2 ** 32 - 1   # along a dimension of a grid


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _pairs(threads):
    """The most workgroups of that many threads."""
    return MOST_THREADS // threads


# (D, type, threads of the rows kernel, of dQ, of dK and dV)
THREADS = [(16, 2, 256, 256, 256), (64, 1, 256, 256, 256), (128, 2, 128, 256, 256), (128, 0, 128, 256, 256), (256, 1, 128, 256, 512),
           (256, 0, 64, 256, 256)]


@pytest.mark.parametrize("D,dtype,rows,dq,dkdv", THREADS)
def test_pairs_of_one_launch(lib, D, dtype, rows, dq, dkdv):
    """One query and one key each: a workgroup to a pair in every kernel."""
    for query, most in ((lib.kv_cross_forward_workspace, _pairs(rows)), (lib.kv_cross_backward_workspace, _pairs(max(dq, dkdv)))):
        assert query(most, 1, 1, 1, 1, D, dtype) >= 0
        assert query(most + 1, 1, 1, 1, 1, D, dtype) == TOO_LARGE
    paged = lib.kv_paged_forward_workspace
    assert paged(_pairs(rows), 1, 1, 1, D, 16, 1, 1, 0, dtype) >= 0
    assert paged(_pairs(rows) + 1, 1, 1, 1, D, 16, 1, 1, 0, dtype) == TOO_LARGE
    if dtype != 0:   # gradients of nothing: zeros for dK and dV
        assert lib.kv_cross_backward_workspace(_pairs(dkdv), 1, 1, 0, 128, D, dtype) >= 0
        assert lib.kv_cross_backward_workspace(_pairs(dkdv), 1, 1, 0, 129, D, dtype) == TOO_LARGE
        assert lib.kv_cross_forward_workspace(_pairs(dkdv), 1, 1, 0, 129, D, dtype) == 0


def test_the_forward_is_not_refused_for_its_backward(lib):
    """One query over many keys: the forward has a workgroup for a run of keys, dK and dV one for 128."""
    sizes = (300, 64, 64, 1, 1 << 20, 16, 2)
    assert lib.kv_cross_backward_workspace(*sizes) == TOO_LARGE
    assert lib.kv_cross_forward_workspace(*sizes) >= 0


def test_calls_say_so_before_they_launch(lib):
    """Null streams and host pointers: a launch would fail with another code, or enqueue dQ alone."""
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    st = (ctypes.c_int64 * 4)(0, 0, 16, 1)

    def forward(B, Tq, Tk):
        return lib.kv_cross_forward(p, p, p, None, 0, None, 0, p, None, p, 1 << 60, st, st, st, B, 1, 1, Tq, Tk, 16, 0.1, 2, None)

    def backward(B, Tq, Tk):
        return lib.kv_cross_backward(p, p, p, None, 0, None, 0, p, p, p, p, p, p, p, 1 << 60, st, st, st, st, st, B, 1, 1, Tq, Tk, 16, 0.1, 2, None)

    for f in (forward, backward):
        assert f(1 << 24, 1, 1) == TOO_LARGE
        assert f(1 << 18, 1 << 13, 1) == TOO_LARGE
    assert backward(1 << 18, 1, 1 << 13) == TOO_LARGE   # dQ alone would fit
    assert lib.kv_paged_forward(p, p, p, p, 1, p, 1, None, 0, p, None, p, 1 << 60, st, st, st, 1 << 24, 1, 1, 1, 16, 4, 16, 1, 1, 0, 0.1, 2,
                                None) == TOO_LARGE


def test_scales_that_float32_does_not_hold(lib):
    """A scale that is finite in Python and not in the kernels gave NaN for every row."""
    q, k = torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 7, 64)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    st = (ctypes.c_int64 * 4)(0, 0, 16, 1)
    for scale in (1e39, -1e300, 2.5e38, float("inf"), float("nan")):
        with pytest.raises(AssertionError, match="sm_scale"):
            ops._validate_cross(q, k, k, None, None, scale)
        with pytest.raises(AssertionError, match="sm_scale"):
            ops._validate_paged(q, k, k, table, lens, 1, 0, scale, None)
        f = min(max(scale, -3.4e38), 3.4e38)   # what a float holds of it (NaN stays)
        assert lib.kv_cross_forward(p, p, p, None, 0, None, 0, p, None, None, 0, st, st, st, 1, 1, 1, 1, 1, 16, f, 2, None) == ARG
        assert lib.kv_cross_backward(p, p, p, None, 0, None, 0, p, p, p, p, p, p, p, 1 << 20, st, st, st, st, st, 1, 1, 1, 1, 1, 16, f, 2, None) == ARG
        assert lib.kv_paged_forward(p, p, p, p, 1, p, 1, None, 0, p, None, None, 0, st, st, st, 1, 1, 1, 1, 16, 4, 16, 1, 1, 0, f, 2, None) == ARG
    ops._validate_cross(q, k, k, None, None, -2.0 ** 127)
    ops._validate_paged(q, k, k, table, lens, 1, 0, 1e38, None)


@pytest.mark.gpu
def test_largest_scales_on_the_gpu():
    """The refusals through the public functions, and the largest scale on scores that it leaves in range: the first key's value, or the
    last one's for a negative scale."""
    from cross_attention import cross_attention
    from paged_attention import paged_attention

    q, k, v = (torch.zeros(1, 1, n, 16, device="cuda:0") for n in (3, 5, 5))
    q[..., 0], k[0, 0, :, 0] = 1.0, torch.tensor([1.0, 0.75, 0.5, 0.25, 0.125])
    v[0, 0] = torch.arange(5.0, device="cuda:0")[:, None]
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda:0"), torch.full((1,), 5, dtype=torch.int32, device="cuda:0")
    for call in (lambda s: cross_attention(q, k, v, sm_scale=s), lambda s: cross_attention(q.expand(1, 1, 3, 16).repeat(1, 1, 30, 1), k, v, sm_scale=s),
                 lambda s: paged_attention(q[:, :, :1], k, v, table, lens, sm_scale=s)):
        assert (call(2.0 ** 127) == 0).all() and (call(-2.0 ** 127) == 4).all()
        for s in (1e39, 2.5e38, -1e300):
            with pytest.raises(AssertionError, match="sm_scale"):
                call(s)
