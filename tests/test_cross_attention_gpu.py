"""Cross attention on the GPU against the float64 oracle, element by element within bounds counted in roundings
(oracle/kv_oracle.py), at the sizes, lengths and layouts where it can go wrong."""
import pytest
import torch

from cross_attention import cross_attention, cross_attention_reference
from oracle import kv_oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _inputs(B, Hq, Hkv, Tq, Tk, D, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype) for s in ((B, Hq, Tq, D), (B, Hkv, Tk, D), (B, Hkv, Tk, D), (B, Hq, Tq, D))]


def _lens(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def _run(q, k, v, d_o, lens, q_lens, scale=None):
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    on = [None if x is None else x.to(DEV) for x in (lens, q_lens)]
    o, lse = cross_attention(*leaves, *on, sm_scale=scale, return_lse=True)
    grads = torch.autograd.grad(o, leaves, d_o.to(DEV))
    return dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *grads)))


def _check(q, k, v, d_o, lens=None, q_lens=None, scale=None):
    lens, q_lens = _lens(lens), _lens(q_lens)
    want = kv_oracle.cross(q, k, v, lens, q_lens, scale, d_o)
    got = _run(q, k, v, d_o, lens, q_lens, scale)
    torch.cuda.synchronize()
    for name in want:
        kv_oracle.assert_within(name, got[name], want[name])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,lens,q_lens", [
    (2, 2, 2, 40, 70, [70, 33], [40, 1]),          # one tile and a part of one
    (3, 4, 2, 150, 200, [1, 0, 200], [150, 7, 0]),   # shared heads, lengths of none and one
    (1, 6, 2, 67, 129, None, None),                # three heads to a key head: rows cross the tiles
])
def test_against_oracle(dtype, D, B, Hq, Hkv, Tq, Tk, lens, q_lens):
    _check(*_inputs(B, Hq, Hkv, Tq, Tk, D, dtype), lens, q_lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,Tq,Tk,lens", [(2, 2, 1, 300, [300, 0]), (8, 2, 1, 1100, [1100, 513]), (4, 2, 7, 37, [1, 36]),
                                               (32, 1, 1, 65, None), (2, 1, 16, 2100, [2100, 31])])
def test_few_rows(dtype, D, Hq, Hkv, Tq, Tk, lens):
    """Up to 32 rows of a key head run a kernel of their own, long keys in shares that are joined."""
    _check(*_inputs(2, Hq, Hkv, Tq, Tk, D, dtype), lens, None if Tq == 1 else [Tq, Tq - 3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_one_token_of_many_lengths(dtype, D):
    """Many sequences, whose parts the workgroups find from the lengths."""
    B, Hq, Hkv, Tk = 72, 8, 4, 3200
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, Tk + 1, (B,), generator=g).to(torch.int32)
    lens[0], lens[1], lens[63], lens[64], lens[-1] = 0, Tk, 1, 2049, 0
    q, k, v, _ = _inputs(B, Hq, Hkv, 1, Tk, D, dtype)
    o, lse = cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), lens.to(DEV), return_lse=True)
    some = [0, 1, 2, 62, 63, 64, 65, B - 1]
    want = kv_oracle.cross(q[some], k[some], v[some], lens[some])
    kv_oracle.assert_within("o", o[some], want["o"])
    kv_oracle.assert_within("lse", lse[some], want["lse"])
    order = torch.randperm(B, generator=g)
    again = cross_attention(q[order].to(DEV), k[order].to(DEV), v[order].to(DEV), lens[order].to(DEV))
    assert torch.equal(again.cpu(), o.cpu()[order])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Tq,Tk,lens,q_lens", [(40, 1500, [1500, 260], None), (1500, 40, [40, 3], [1300, 1500]),
                                               (700, 900, [900, 0], [1, 700])])
def test_split_work(dtype, D, Tq, Tk, lens, q_lens):
    """Few workgroups: the keys (for dK and dV the rows) are divided and float32 parts added up."""
    from kv_attention import _lib

    dt = DTYPES.index(dtype)
    plain = 2 * ((4 * 2 * Tq * 4 + 255) // 256 * 256)   # lse and delta of all rows
    assert _lib.load().kv_cross_backward_workspace(2, 4, 2, Tq, Tk, D, dt) > plain
    _check(*_inputs(2, 4, 2, Tq, Tk, D, dtype), lens, q_lens)


@pytest.mark.parametrize("dtype,B,Hq,Hkv,Tq,Tk,D,lens,q_lens", [
    (torch.float16, 2, 8, 8, 1300, 1100, 64, [1100, 40], [1300, 3]),      # more workgroups than half of the CUs, a place for each share
    (torch.bfloat16, 2, 8, 8, 1100, 1300, 128, [1300, 1025], None),
    (torch.float32, 1, 8, 4, 1200, 1100, 32, None, [1111]),
    (torch.float16, 5, 2, 1, 3000, 15, 32, [15, 1, 0, 9, 15], [3000, 1, 700, 0, 2999]),
    (torch.bfloat16, 3, 8, 8, 1400, 6500, 64, [6500, 64, 6401], [1400, 1300, 127]),   # more than CUs, long runs
    (torch.float16, 2, 8, 2, 512, 3300, 256, [3300, 3201], None),
])
def test_divided_runs(dtype, B, Hq, Hkv, Tq, Tk, D, lens, q_lens):
    """Every rule by which runs are divided, against the oracle on one key head of each batch entry."""
    from kv_attention import _lib

    q, k, v, d_o = _inputs(B, Hq, Hkv, Tq, Tk, D, dtype)
    lens, q_lens = _lens(lens), _lens(q_lens)
    plain = 2 * ((B * Hq * Tq * 4 + 255) // 256 * 256)
    assert _lib.load().kv_cross_backward_workspace(B, Hq, Hkv, Tq, Tk, D, DTYPES.index(dtype)) > plain
    got = _run(q, k, v, d_o, lens, q_lens)
    torch.cuda.synchronize()
    G = Hq // Hkv
    for b in range(B):
        h = b % Hkv
        heads = slice(h * G, (h + 1) * G)
        one = [t[b:b + 1] for t in (q[:, heads], k[:, h:h + 1], v[:, h:h + 1], d_o[:, heads])]
        want = kv_oracle.cross(*one[:3], None if lens is None else lens[b:b + 1], None if q_lens is None else q_lens[b:b + 1], None, one[3])
        for name in want:
            of = slice(h, h + 1) if name in ("dk", "dv") else heads
            kv_oracle.assert_within(f"{name} of {b}", got[name][b:b + 1, of], want[name])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,lens,q_lens,layout", [
    (8, 16, 16, 500, 520, [520, 64, 0, 1, 519, 300, 128, 65], [500, 1, 500, 0, 257, 256, 64, 333], "plain"),
    (4, 32, 8, 512, 1100, [1100, 513, 64, 0], None, "plain"),           # heads of a key head as one run of rows
    (4, 32, 8, 512, 1100, [1100, 513, 64, 0], [512, 500, 3, 512], "plain"),   # padding inside them: dK and dV of the tile kernel
    (4, 32, 8, 512, 1100, None, None, "tokens"),                        # heads next to each other: likewise
    (2, 8, 8, 600, 2100, [2100, 1999], [600, 77], "plain"),             # dK and dV by hand, too few workgroups for the others
    (8, 64, 1, 256, 600, None, None, "plain"),                          # the reverse
])
def test_hand_scheduled(dtype, B, Hq, Hkv, Tq, Tk, lens, q_lens, layout):
    """Head dimension 128 on long runs, against the oracle on some heads and the tile kernels' bounds."""
    D = 128
    q, k, v, d_o = _inputs(B, Hq, Hkv, Tq, Tk, D, dtype)
    lens, q_lens = _lens(lens), _lens(q_lens)
    on = [t.to(DEV) for t in (q, k, v, d_o)]
    if layout == "tokens":
        on = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in on]
    leaves = [t.requires_grad_() for t in on[:3]]
    args = [None if x is None else x.to(DEV) for x in (lens, q_lens)]
    o, lse = cross_attention(*leaves, *args, return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, leaves, on[3])
    torch.cuda.synchronize()
    G = Hq // Hkv
    for b in range(B):
        h = b % Hkv
        heads = slice(h * G, (h + 1) * G)
        one = [t[b:b + 1] for t in (q[:, heads], k[:, h:h + 1], v[:, h:h + 1], d_o[:, heads])]
        want = kv_oracle.cross(*one[:3], None if lens is None else lens[b:b + 1], None if q_lens is None else q_lens[b:b + 1], None, one[3])
        for name, got in (("o", o[b:b + 1, heads]), ("lse", lse[b:b + 1, heads]), ("dq", dq[b:b + 1, heads]),
                          ("dk", dk[b:b + 1, h:h + 1]), ("dv", dv[b:b + 1, h:h + 1])):
            kv_oracle.assert_within(f"{name} of {b}", got, want[name])


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_hand_scheduled_padding_is_never_used(junk):
    B, H, Tq, Tk = 8, 16, 500, 600
    q, k, v, d_o = _inputs(B, H, H, Tq, Tk, 128, torch.bfloat16)
    lens, q_lens = [600, 1, 64, 65, 0, 333, 512, 599], [500, 499, 256, 257, 31, 1, 0, 64]
    clean = _run(q, k, v, d_o, _lens(lens), _lens(q_lens))
    for b in range(B):
        k[b, :, lens[b]:], v[b, :, lens[b]:] = junk, junk
        q[b, :, q_lens[b]:], d_o[b, :, q_lens[b]:] = junk, junk
    dirty = _run(q, k, v, d_o, _lens(lens), _lens(q_lens))
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    assert (dirty["lse"][4, :, :31] == -float("inf")).all() and not dirty["o"][4].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [None, -0.2])
@pytest.mark.parametrize("Hq,Hkv,Tq,Tk,D", [(12, 12, 300, 65, 32), (4, 4, 300, 65, 256), (8, 2, 90, 300, 64), (16, 16, 500, 520, 128)])
def test_few_keys(dtype, scale, Hq, Hkv, Tq, Tk, D):
    """Gradients of rows over few keys carry the roundings of dS and of the result only, not that of O.  A rounding is uniform over half a
    step u to either side: relative to a value with any mantissa its root mean square is u sqrt(mean(1 / m^2) / 3) = 0.425 u, two of them
    0.60 u.  Over one key dS is 0: P, a sum of which is 1 within 2^-19, leaves that much of dP."""
    lens = [1, 2, 3, 5, 8, 20, 33, 64]
    q, k, v, d_o = _inputs(8, Hq, Hkv, Tq, Tk, D, dtype)
    got = _run(q, k, v, d_o, _lens(lens), None, scale)
    torch.cuda.synchronize()
    u = torch.finfo(dtype).eps / 2
    s = abs(D ** -0.5 if scale is None else scale)
    for b, n in enumerate(lens):
        one = [t[b:b + 1].double() for t in (q, k[:, :, :n], v[:, :, :n], d_o)]
        leaves = [t.requires_grad_() for t in one[:3]]
        want = torch.autograd.grad(cross_attention_reference(*leaves, sm_scale=scale)[0], leaves, one[3])
        if n == 1:
            heads = [t.repeat_interleave(Hq // Hkv, dim=1) for t in one[1:3]]
            dp = (one[3].abs() @ heads[1].abs().transpose(-1, -2)) * 2.0 ** -18
            assert (got["dq"][b].cpu().double().abs() <= s * dp[0] * heads[0][0].abs() + 2.0 ** -24).all()
            continue
        for name, x, w in (("dq", got["dq"][b], want[0][0]), ("dk", got["dk"][b, :, :n], want[1][0])):
            assert (x.cpu().double() - w).norm() <= 0.66 * u * w.norm(), (name, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.7])
def test_scales(dtype, scale):
    q, k, v, d_o = _inputs(1, 2, 1, 70, 90, 64, dtype)
    _check(q * 0.5, k * 0.5, v, d_o, scale=scale)
    _check(q[:, :, :5] * 0.5, k * 0.5, v, d_o[:, :, :5], scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [3, 100])
def test_large_scores(dtype, Tq):
    """Scores whose exponentials pass every range, with a maximum that keeps moving."""
    q, k, v, d_o = _inputs(1, 1, 1, Tq, 333, 64, dtype)
    k = (k.float() * torch.linspace(0.1, 8, 333)[:, None]).to(dtype)
    _check(q, k, v, d_o)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [5, 140])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_padding_is_never_used(dtype, Tq, D, junk):
    q, k, v, d_o = _inputs(3, 4, 2, Tq, 150, D, dtype)
    lens, q_lens = [150, 41, 0], [Tq - 2, Tq, 3]
    clean = _run(q, k, v, d_o, _lens(lens), _lens(q_lens))
    for b in range(3):
        k[b, :, lens[b]:], v[b, :, lens[b]:] = junk, junk
        q[b, :, q_lens[b]:], d_o[b, :, q_lens[b]:] = junk, junk
    dirty = _run(q, k, v, d_o, _lens(lens), _lens(q_lens))
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    for b in range(3):
        assert not dirty["o"][b, :, q_lens[b]:].any() and not dirty["dq"][b, :, q_lens[b]:].any()
        assert not dirty["lse"][b, :, q_lens[b]:].any()
        assert not dirty["dk"][b, :, lens[b]:].any() and not dirty["dv"][b, :, lens[b]:].any()
    assert (dirty["lse"][2, :, :3] == -float("inf")).all() and not dirty["o"][2].any() and not dirty["dq"][2].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 33), (130, 1), (0, 40), (40, 0), (1, 0)])
def test_smallest(dtype, Tq, Tk):
    got = _check(*_inputs(2, 2, 1, Tq, Tk, 64, dtype))
    if Tk == 0:
        assert not got["o"].any() and (got["lse"] == -float("inf")).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("Tq", [6, 90])
def test_strides(dtype, Tq):
    """Views of projection outputs, broadcast heads and batch entries, strides that have to be copied."""
    B, H, Tk, D = 2, 4, 120, 64
    g = torch.Generator().manual_seed(8)
    kv = torch.randn(B, Tk, 2, H, D, generator=g).to(dtype).to(DEV)
    qs = torch.randn(B, Tq, H, D, generator=g).to(dtype).to(DEV)
    d_o = torch.randn(B, Tq, H, D, generator=g).to(dtype).to(DEV)
    wide = torch.randn(B, H, Tk, D + 1, generator=g).to(dtype).to(DEV)
    one = torch.randn(1, 1, Tk, D, generator=g).to(dtype).to(DEV)
    lens = torch.tensor([[120, 7], [33, 9]], dtype=torch.int32, device=DEV)[:, 0]
    for k, v in ((kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)), (wide[..., 1:], wide[..., :-1]),
                 (one.expand(B, H, Tk, D), one.expand(B, H, Tk, D)), (wide[:, :2, :, :D], wide[:, :2, ::1, 1:])):
        q = qs.transpose(1, 2)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        grads = torch.autograd.grad(cross_attention(*leaves, lens), leaves, d_o.transpose(1, 2))
        plain = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*plain, lens.contiguous())
        for a, b in zip(grads, torch.autograd.grad(out, plain, d_o.transpose(1, 2).contiguous())):
            assert torch.equal(a, b)
        assert torch.equal(out, cross_attention(*leaves, lens))


def test_gradients_are_those_of_differences():
    """Directional derivatives of the float32 forward against the gradients."""
    q, k, v, d_o = (t.to(DEV) for t in _inputs(2, 4, 2, 45, 60, 32, torch.float32))
    lens, q_lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([60, 31], [45, 20]))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves, lens, q_lens), leaves, d_o)
    g = torch.Generator().manual_seed(9)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=g).to(DEV)
        h = 2.0 ** -6
        side = []
        for sign in (1, -1):
            moved = [t + sign * h * step if j == i else t for j, t in enumerate((q, k, v))]
            side.append((cross_attention(*moved, lens, q_lens).double() * d_o.double()).sum())
        slope, want = (side[0] - side[1]) / (2 * h), (grads[i].double() * step.double()).sum()
        # third derivatives, h^2 / 6 of them, and the float32 rounding of about 8000 outputs, divided by 2 h
        assert abs(slope - want) <= 2e-3 * abs(want) + 0.5


def test_matches_the_plain_reference():
    q, k, v, _ = (t.to(DEV) for t in _inputs(2, 4, 2, 50, 60, 64, torch.float32))
    lens, q_lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([60, 0], [50, 20]))
    want, valid = cross_attention_reference(q, k, v, lens, q_lens)
    got = cross_attention(q, k, v, lens, q_lens)
    assert (got - want).abs().max() < 1e-4 and not got[~valid.expand_as(got)].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_from_call_to_call(dtype):
    q, k, v, d_o = _inputs(4, 8, 2, 200, 1000, 64, dtype)
    first, second = (_run(q, k, v, d_o, _lens([1000, 5, 600, 999]), None) for _ in range(2))
    for name in first:
        assert torch.equal(first[name], second[name]), name


@pytest.mark.parametrize("Tq", [1, 100])
def test_backward_without_the_log_sum_exp(Tq):
    q, k, v, d_o = (t.to(DEV) for t in _inputs(2, 4, 2, Tq, 70, 64, torch.bfloat16))
    op = torch.ops.alexdremov_cross_attention
    o, lse = op.forward(q, k, v, None, None, 0.125, True)
    _, none = op.forward(q, k, v, None, None, 0.125, False)
    assert none.numel() == 0
    for a, b in zip(op.backward(q, k, v, None, None, o, lse, d_o, 0.125), op.backward(q, k, v, None, None, o, none, d_o.float(), 0.125)):
        assert torch.equal(a, b)


def test_graph_replays():
    """Forward and backward captured once and replayed on new values, with eager work in between, on two workspaces."""
    shapes = [_inputs(2, 4, 2, 40, 1500, 64, torch.bfloat16, seed) for seed in (1, 2, 3)]
    static = [t.to(DEV) for t in shapes[0]]
    lens = torch.tensor([1500, 700], dtype=torch.int32, device=DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in static[:3]]
        o = cross_attention(*leaves, lens)
        few = cross_attention(static[0][:, :, :2].detach(), static[1], static[2], lens)
        return (o.detach(), few, *torch.autograd.grad(o, leaves, static[3]))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for values in shapes + shapes[:1]:
        for s, x in zip(static, values):
            s.copy_(x.to(DEV))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_streams():
    """Calls on two streams at once, each with workspaces of its own."""
    sets = [[t.to(DEV) for t in _inputs(2, 4, 2, 40, 3000, 64, torch.float16, seed)] for seed in (1, 2)]

    def both(x):
        leaves = [t.detach().requires_grad_() for t in x[:3]]
        o = cross_attention(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, x[3]))

    want = [both(x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i].append(both(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_opcheck():
    q, k, v, _ = (t.to(DEV) for t in _inputs(2, 4, 2, 40, 70, 64, torch.float32))
    lens = torch.tensor([70, 20], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    torch.library.opcheck(torch.ops.alexdremov_cross_attention.forward.default, (*leaves, lens, None, 0.125, True))
    out = torch.compile(cross_attention, backend="aot_eager", fullgraph=True)(*leaves, lens)
    assert torch.equal(out, cross_attention(*leaves, lens))
    for a, b in zip(torch.autograd.grad(out.sum(), leaves), torch.autograd.grad(cross_attention(*leaves, lens).sum(), leaves)):
        assert torch.equal(a, b)


def test_long_rows_of_keys():
    """Strides that the 32-bit offsets of one head do not hold are copied."""
    T, D = 70, 64
    g = torch.Generator().manual_seed(4)
    base = torch.zeros(T, (1 << 31) // 70 // 8 * 8, dtype=torch.float16, device=DEV)   # 4 GiB
    k = torch.randn(T, D, generator=g).half()
    base[:, :D] = k.to(DEV)
    strided = base[:, :D][None, None]
    q = torch.randn(1, 1, 40, D, generator=g).half().to(DEV)
    assert (T + 1024) * strided.stride(2) * 2 >= 1 << 32
    plain = k.to(DEV)[None, None]
    assert torch.equal(cross_attention(q, strided, strided), cross_attention(q, plain, plain))
