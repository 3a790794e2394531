"""Sizes at the limits of a launch, on the host: refused by name before anything is enqueued, and one workgroup below them not."""
import ctypes

import pytest

from kv_attention import _lib

TOO_LARGE = -5
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
