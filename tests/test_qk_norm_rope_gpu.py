"""Norms and rotation of queries and keys on the GPU, forward and backward, against the float64 oracle within bounds counted in roundings,
against differences, in strided layouts, captured, and before the attention that takes them."""
import pytest
import torch

from cross_attention import cross_attention
from kv_attention import _lib
from oracle import kv_oracle
from qk_norm_rope import qk_norm_rope, qk_norm_rope_reference
from streaming_attention import streaming_attention

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _tables(n, rot, base=10000.0):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return angle.cos().float(), angle.sin().float()


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype)


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def _dev(t):
    return None if t is None else t.to(DEV)


def _check(q, k, cos, sin, wq=None, wk=None, lens=None, positions=None, eps=None, interleaved=False, seed=3):
    """Forward and backward of CPU tensors against the oracle."""
    B, _, T, D = q.shape
    g = torch.Generator().manual_seed(seed)
    grads = [_randn(g, x.dtype, *x.shape) for x in (q, k)]
    leaves = [None if t is None else t.to(DEV).requires_grad_() for t in (q, k, wq, wk)]
    out = qk_norm_rope(leaves[0], leaves[1], _dev(cos), _dev(sin), leaves[2], leaves[3], _dev(lens), _dev(positions), eps, interleaved)
    there = [t for t in leaves if t is not None]
    got = torch.autograd.grad(out, there, [_dev(t) for t in grads])
    torch.cuda.synchronize()
    at = torch.arange(T).expand(B, T) if positions is None else positions.long()
    live = (at >= 0) & (at < cos.shape[0])
    if lens is not None:
        live &= torch.arange(T) < lens.clamp(0, T)[:, None]
    for i, (x, w, name) in enumerate(((q, wq, "q"), (k, wk, "k"))):
        mask = live[:, None].expand(B, x.shape[1], T)
        angles = [t[at.clamp(0, cos.shape[0] - 1)][:, None].expand(B, x.shape[1], T, -1)[mask] for t in (cos, sin)]
        want = kv_oracle.rope_rows(x[mask], *angles, w, eps, interleaved, grads[i][mask])
        for what, have in (("out", out[i]), ("dx", got[i])):
            assert have.is_contiguous() and have.dtype == x.dtype
            full = [torch.zeros(x.shape, dtype=torch.float64) for _ in range(2)]
            for part, value in zip(full, want[what]):
                part[mask] = value
            kv_oracle.assert_within(f"{what} of {name}", have, tuple(full))
        if w is not None:
            have = got[2 + (i if wq is not None else 0)]
            assert have.dtype == w.dtype
            kv_oracle.assert_within(f"weights of {name}", have, want["dw"])
    return out, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot,eps,f32", [("all", 1e-6, False), ("all", None, False), ("some", 1e-5, True), ("16", 1e-2, False)])
def test_head_dims(dtype, D, interleaved, rot, eps, f32):
    rot = {"all": D, "some": max(16, D // 2 + D // 4 // 16 * 16), "16": 16}[rot]
    g = torch.Generator().manual_seed(D)
    q, k = _randn(g, dtype, 2, 6, 37, D), _randn(g, dtype, 2, 2, 37, D)
    wq, wk = ((1 + 0.3 * _randn(g, torch.float32, D)).to(torch.float32 if f32 else dtype) for _ in range(2)) if eps is not None else (None, None)
    _check(q, k, *_tables(37, rot), wq, wk, eps=eps, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,T", [(1, 1, 1, 1), (3, 5, 3, 1), (1, 40, 8, 2), (2, 9, 1, 333), (1, 3, 17, 1000), (700, 1, 1, 1), (1, 64, 8, 301)])
def test_sizes(dtype, B, Hq, Hkv, T):
    g = torch.Generator().manual_seed(T)
    wq, wk = (1 + 0.3 * _randn(g, torch.float32, 64) for _ in range(2))
    _check(_randn(g, dtype, B, Hq, T, 64), _randn(g, dtype, B, Hkv, T, 64), *_tables(T, 64), wq.to(dtype), wk.to(dtype), eps=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weights", ["q", "k", "none"])
def test_some_weights(dtype, weights):
    g = torch.Generator().manual_seed(4)
    w = {n: (1 + 0.3 * _randn(g, torch.float32, 32)).to(dtype) if n == weights else None for n in "qk"}
    _check(_randn(g, dtype, 2, 4, 50, 32), _randn(g, dtype, 2, 2, 50, 32), *_tables(50, 32), w["q"], w["k"], eps=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,positions", [([50, 0, 13], None), (None, "far"), ([50, 7, -3], "outside"), ([99, 49, 1], "shared")])
def test_padding_and_positions(dtype, lens, positions):
    """Lengths of zero and beyond, positions far out, outside the table, of another order; what stands in padding does not matter."""
    g = torch.Generator().manual_seed(5)
    B, T, D, rows = 3, 50, 64, 100000
    cos, sin = _tables(rows, D)
    at = None
    if positions == "far":
        at = torch.randint(0, rows, (B, T), generator=g, dtype=torch.int32)
    elif positions == "outside":
        at = torch.randint(-50, 50, (B, T), generator=g, dtype=torch.int32)
        at[1, 3], at[1, 4], at[0, 0], at[0, 1] = rows, rows - 1, -2 ** 31, 2 ** 31 - 1
    elif positions == "shared":
        at = torch.arange(T, 0, -1, dtype=torch.int32)[None].expand(B, T)
    q, k = _randn(g, dtype, B, 4, T, D), _randn(g, dtype, B, 2, T, D)
    w = (1 + 0.3 * _randn(g, torch.float32, D)).to(dtype)
    out, grads = _check(q, k, cos, sin, w, w, _i32(lens), at, 1e-6)
    live = torch.ones(B, T, dtype=torch.bool) if at is None else (at >= 0) & (at < rows)
    if lens is not None:
        live = live & (torch.arange(T) < _i32(lens)[:, None])
    dead = ~live[:, None, :, None]
    q, k = (torch.where(dead, float("nan"), x) for x in (q, k))
    again = _check(q, k, cos, sin, w, w, _i32(lens), at, 1e-6)
    for a, b in zip((*out, *grads), (*again[0], *again[1])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tables_without_rows(dtype):
    q, k = (torch.randn(2, h, 5, 32, device=DEV).to(dtype).requires_grad_() for h in (4, 2))
    w = torch.ones(32, device=DEV, dtype=dtype, requires_grad=True)
    empty = torch.zeros(0, 16, device=DEV)
    out = qk_norm_rope(q, k, empty, empty, w, w)
    grads = torch.autograd.grad(out, (q, k, w), [torch.ones_like(t) for t in out])
    assert not any(t.any() for t in (*out, *grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 128])
def test_layouts(dtype, D):
    """Views of a projection's output, reversed heads, expanded batches, rows that are not aligned: the same bits as contiguous ones."""
    g = torch.Generator().manual_seed(6)
    B, Hq, Hkv, T = 3, 6, 2, 41
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    w = (1 + 0.3 * _randn(g, torch.float32, D)).to(dtype).to(DEV)
    d = [_randn(g, dtype, B, h, T, D).to(DEV) for h in (Hq, Hkv)]

    def step(q, k, grads, cos=cos, sin=sin, wq=w):
        leaves = [t.detach().requires_grad_() for t in (q, k, wq)]
        out = qk_norm_rope(leaves[0], leaves[1], cos, sin, leaves[2], leaves[2])
        return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, grads))

    qkv = _randn(g, dtype, B, T, Hq + 2 * Hkv, D).to(DEV).transpose(1, 2)
    views = [(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv])]
    wide = _randn(g, dtype, B, Hq + Hkv, T, D + 24).to(DEV)
    views.append((wide[:, :Hq, :, 8:8 + D], wide[:, Hq:, :, 8:8 + D]))            # 16-byte steps
    odd = _randn(g, dtype, B, Hq + Hkv, T, D + 3).to(DEV)
    views.append((odd[:, :Hq, :, 1:1 + D], odd[:, Hq:, :, 3:3 + D]))              # neither address nor steps
    one = _randn(g, dtype, 1, Hq + Hkv, 1, D).to(DEV).expand(B, Hq + Hkv, T, D)
    views.append((one[:, :Hq], one[:, Hq:]))
    views.append((qkv[:, :Hq].transpose(0, 1).contiguous().transpose(0, 1), qkv[:, -Hkv:]))
    for q, k in views:
        want = step(q.contiguous(), k.contiguous(), d)
        got = step(q, k, d)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        spread = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in d]
        assert all(torch.equal(a, b) for a, b in zip(step(q, k, spread), want))
        tables = [torch.cat([t, t], 1)[:, :D // 2] for t in (cos, sin)]
        assert all(torch.equal(a, b) for a, b in zip(step(q, k, d, *tables), want))
        tables = [torch.cat([t[:, :1], t], 1)[:, 1:] for t in (cos, sin)]          # not aligned
        assert all(torch.equal(a, b) for a, b in zip(step(q, k, d, *tables, torch.stack([w, w], 1)[:, 0]), want))


def test_against_differences():
    """Float32 gradients against central differences of a float64 sum of the reference's outputs."""
    g = torch.Generator().manual_seed(7)
    q, k, w = _randn(g, torch.float64, 1, 2, 5, 32), _randn(g, torch.float64, 1, 1, 5, 32), 1 + 0.3 * _randn(g, torch.float64, 32)
    q, k, w = (t.float().double() for t in (q, k, w))   # what float32 holds
    cos, sin = _tables(5, 16)
    up = [_randn(g, torch.float32, *t.shape).double() for t in (q, k)]

    def total(q, k, w):
        return sum((a * b).sum() for a, b in zip(qk_norm_rope_reference(q, k, cos.double(), sin.double(), w, w), up))

    leaves = [t.float().to(DEV).requires_grad_() for t in (q, k, w)]
    out = qk_norm_rope(leaves[0], leaves[1], cos.to(DEV), sin.to(DEV), leaves[2], leaves[2])
    grads = torch.autograd.grad(out, leaves, [t.float().to(DEV) for t in up])
    step = 1e-5
    for i, (x, got) in enumerate(zip((q, k, w), grads)):
        for at in range(0, x.numel(), 7):
            moved = [t.clone() for t in (q, k, w)]
            moved[i].view(-1)[at] += step
            high = total(*moved)
            moved[i].view(-1)[at] -= 2 * step
            slope = float(high - total(*moved)) / (2 * step)
            # differences: their own rounding 1e-16 * 300 / step and third derivatives times step^2; float32: 100 roundings of sums below 50
            assert abs(float(got.view(-1)[at]) - slope) <= 1e-7 + 100 * 2.0 ** -24 * 50


@pytest.mark.parametrize("dtype", DTYPES)
def test_magnitudes(dtype):
    """Rows of zeros, of tiny and of large values."""
    g = torch.Generator().manual_seed(8)
    q, k = _randn(g, dtype, 1, 4, 40, 64), _randn(g, dtype, 1, 2, 40, 64)
    big = 1e4 if dtype == torch.float16 else 1e15
    small = 1e-6 if dtype == torch.float16 else 1e-15
    for x in (q, k):
        x[:, 0] = 0
        x[:, 1, ::2] *= big if dtype != torch.float16 else 1e3
        x[:, 1, 1::2] *= small
    w = (1 + 0.3 * _randn(g, torch.float32, 64)).to(dtype)
    _check(q, k, *_tables(40, 64), w, w, eps=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite_stay_in_their_pair(dtype):
    """Without norms a channel past the rotated ones keeps what it holds, and its neighbours keep theirs."""
    g = torch.Generator().manual_seed(9)
    x = _randn(g, dtype, 1, 2, 3, 64)
    x[0, 0, 1, 40], x[0, 0, 1, 5] = float("inf"), float("nan")
    for interleaved in (False, True):
        out = qk_norm_rope(x.to(DEV), x.to(DEV), *(t.to(DEV) for t in _tables(3, 32)), eps=None, interleaved=interleaved)[0].cpu()
        bad = torch.nonzero(~torch.isfinite(out[0])).tolist()
        pair = (4, 5) if interleaved else (5, 21)
        assert bad == [[0, 1, pair[0]], [0, 1, pair[1]], [0, 1, 40]]


SHAPES = [(torch.float32, 2, 4, 4, 50, 64), (torch.bfloat16, 2, 32, 8, 500, 128), (torch.float16, 64, 12, 12, 1, 64), (torch.bfloat16, 3, 8, 2, 2000, 256)]


def _step(x, tables, lens):
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = qk_norm_rope(leaves[0], leaves[1], *tables, leaves[2], leaves[3], lens)
    return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, x[4:]))


@pytest.mark.parametrize("shape", SHAPES)
def test_two_graphs(shape):
    """Two captures of forward and backward, replayed in turn, on two streams at once and with eager calls between."""
    dtype, B, Hq, Hkv, T, D = shape
    tables = [t.to(DEV) for t in _tables(T, D)]
    lens = torch.arange(T - B + 1, T + 1, dtype=torch.int32).clamp(min=1).to(DEV)

    def tensors(seed):
        g = torch.Generator().manual_seed(seed)
        return [_randn(g, dtype, *s).to(DEV) for s in ((B, Hq, T, D), (B, Hkv, T, D), (D,), (D,), (B, Hq, T, D), (B, Hkv, T, D))]

    static, fresh = [tensors(s) for s in (1, 2)], [tensors(s) for s in (3, 4)]
    _step(static[0], tables, lens)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(x, tables, lens))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for values in (static, fresh, fresh):
        values = [[t.clone() for t in x] for x in values]
        want = [_step(x, tables, lens) for x in values]
        for s, x in zip(static, values):
            for a, b in zip(s, x):
                a.copy_(b)
        for graph, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_missing_and_foreign_gradients():
    """Only one of the outputs is used; a gradient in another type."""
    g = torch.Generator().manual_seed(10)
    q, k, w = (_randn(g, torch.bfloat16, *s).to(DEV).requires_grad_() for s in ((2, 4, 9, 64), (2, 2, 9, 64), (64,)))
    tables = [t.to(DEV) for t in _tables(9, 64)]
    out = qk_norm_rope(q, k, *tables, w, w)
    dq, dk, dw = torch.autograd.grad(out[0].float().square().sum(), (q, k, w), retain_graph=True)
    assert dq.any() and dw.any() and not dk.any()
    up = out[1].detach().double()
    same = torch.autograd.grad(out[1], (k, w), out[1].detach(), retain_graph=True)
    from_double = torch.ops.alexdremov_qk_norm_rope.backward(torch.zeros_like(out[0]).double(), up, q, k, *tables, w, w, None, None, 1e-6, False, True)
    assert torch.equal(from_double[1], same[0]) and torch.equal(from_double[3].detach(), same[1])


def test_opcheck():
    g = torch.Generator().manual_seed(12)
    q, k, w = (_randn(g, torch.float32, *s).to(DEV).requires_grad_() for s in ((2, 4, 9, 32), (2, 2, 9, 32), (32,)))
    tables = [t.to(DEV) for t in _tables(9, 32)]
    torch.library.opcheck(torch.ops.alexdremov_qk_norm_rope.forward, (q, k, *tables, w, w, None, None, 1e-6, False))
    torch.library.opcheck(torch.ops.alexdremov_qk_norm_rope.forward, (q, k, *tables, None, None, _i32([9, 3]).to(DEV), None, None, True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_before_attention(dtype):
    """A training step as a model makes it: norms, rotation and streaming attention, or cross attention, their gradients against the
    references in float64.  Bounds: the attention's operands are rounded turned rows, each off by half a step."""
    g = torch.Generator().manual_seed(13)
    B, H, T, D = 2, 4, 65, 64
    qkv = _randn(g, dtype, B, T, 3 * H, D)
    w = (1 + 0.2 * _randn(g, torch.float32, D)).to(dtype)
    tables = _tables(T, D)
    lens = _i32([T, 40])
    d_o = _randn(g, dtype, B, H, T, D)

    def step(dev, kind, work):
        x, weight = (t.to(dev).to(work).requires_grad_() for t in (qkv, w))
        heads = x.transpose(1, 2)
        q, k, v = heads[:, :H], heads[:, H:2 * H], heads[:, 2 * H:]
        if kind == "reference":
            q, k = qk_norm_rope_reference(q, k, *[t.to(work) for t in tables], weight, weight, lens)
            at = torch.arange(T)
            gap = at[:, None] // 16 - at // 16
            seen = (gap >= 0) & (gap <= 2) & (at < lens[:, None, None]) & (at < lens[:, None])[:, :, None]
            s = (q @ k.transpose(-1, -2)) * D ** -0.5
            s = s.masked_fill(~seen[:, None], float("-inf"))
            p = torch.softmax(torch.where(seen.any(-1)[:, None, :, None], s, 0.0), -1)
            o = torch.where(seen.any(-1)[:, None, :, None], p @ v, 0.0)
        else:
            q, k = qk_norm_rope(q, k, *[t.to(dev) for t in tables], weight, weight, lens.to(dev))
            o = streaming_attention(q, k, v, lens.to(dev), 16, 2)
        return o.detach(), *torch.autograd.grad(o, (x, weight), d_o.to(dev).to(work))

    want = step("cpu", "reference", torch.float64)
    got = step(DEV, "own", dtype)
    u = kv_oracle.HALF_STEP[dtype] if dtype != torch.float32 else 2.0 ** -20
    for name, a, b in zip(("o", "dx", "dw"), got, want):
        # q, k, P, dS, o, dO's products: some tens of half steps of values of the tensor's own size
        scale = b.abs().amax(-1, keepdim=True).clamp(min=b.abs().mean()) if name != "dw" else b.abs().max()
        assert ((a.double().cpu() - b).abs() <= 40 * u * scale).all(), name


def test_cross_attention_takes_them():
    g = torch.Generator().manual_seed(14)
    q, k, v = (_randn(g, torch.bfloat16, 2, h, 33, 64).to(DEV) for h in (8, 2, 2))
    tables = [t.to(DEV) for t in _tables(33, 64)]
    lens = _i32([33, 20]).to(DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    turned = qk_norm_rope(q, k, *tables, lens=lens)
    o = cross_attention(*turned, v, lens, lens)
    grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
    inner = [t.detach().requires_grad_() for t in turned]
    o2 = cross_attention(*inner, v, lens, lens)
    mid = torch.autograd.grad(o2, inner, torch.ones_like(o))
    want = torch.autograd.grad(qk_norm_rope(q, k, *tables, lens=lens), (q, k), mid)
    assert torch.equal(o, o2) and torch.equal(grads[0], want[0]) and torch.equal(grads[1], want[1])
    assert not grads[0][1, :, 20:].any() and not grads[1][1, :, 20:].any()


def test_another_stream_and_threads():
    import threading

    work = []
    for i, (dtype, B, Hq, Hkv, T, D) in enumerate(SHAPES):
        g = torch.Generator().manual_seed(20 + i)
        x = [_randn(g, dtype, *s).to(DEV) for s in ((B, Hq, T, D), (B, Hkv, T, D), (D,), (D,), (B, Hq, T, D), (B, Hkv, T, D))]
        work.append((x, [t.to(DEV) for t in _tables(T, D)]))
    want = [_step(x, t, None) for x, t in work]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = _step(*work[i], None)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_smallest_eps():
    """Rows of zeros over a subnormal eps: zeros, and gradients of g w / sqrt(eps)."""
    q, k = (torch.zeros(1, h, 3, 64, device=DEV, requires_grad=True) for h in (2, 1))
    cos, sin = torch.ones(3, 32, device=DEV), torch.zeros(3, 32, device=DEV)
    for eps in (2.0 ** -126, 2.0 ** -140, 2.0 ** -148):
        out = qk_norm_rope(q, k, cos, sin, eps=eps)
        assert all(torch.equal(t, torch.zeros_like(t)) for t in out)
        for grad in torch.autograd.grad(out, (q, k), [torch.ones_like(t) for t in out]):
            # the root and three products with it: a few roundings of float32
            assert ((grad.double() * eps ** 0.5 - 1).abs() <= 8 * 2.0 ** -24).all()


def test_weights_without_rows():
    """No sequence, token or head: the C entry leaves zeros in the weights' gradients."""
    lib = _lib.load()
    w = torch.ones(64, device=DEV)
    for B, Hq, Hkv, T in ((0, 2, 1, 8), (2, 2, 1, 0), (2, 0, 0, 8)):
        got = [torch.full((64,), 7.0, device=DEV) for _ in range(2)]
        rc = lib.kv_qk_norm_rope_backward(None, None, None, None, None, None, 0, 0, w.data_ptr(), w.data_ptr(), 1, None, 0, None, None, None, None,
                                          got[0].data_ptr(), got[1].data_ptr(), None, 0, None, None, None, None, B, Hq, Hkv, T, 64, 64, 0, 0, 1e-6,
                                          2, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and all(torch.equal(t, torch.zeros_like(t)) for t in got)


@pytest.mark.parametrize("dtype,D,rot,interleaved", [
    (torch.bfloat16, 256, 128, False), (torch.float16, 256, 64, False), (torch.float32, 128, 64, False), (torch.float16, 128, 128, False),
    (torch.bfloat16, 128, 64, False), (torch.bfloat16, 128, 32, True), (torch.float32, 64, 64, False), (torch.float16, 256, 256, True)])
def test_large_calls_give_what_small_ones_give(dtype, D, rot, interleaved):
    """More than the caches hold, with stores past them where a store covers whole lines: the same bits as in pieces, forward and backward."""
    B, H = 2, 16
    T = (20 << 20) // (B * (H + 2) * D * dtype.itemsize) + 3
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k = (torch.randn(B, h, T, D, generator=g, device=DEV).to(dtype).requires_grad_() for h in (H, 2))
    up = [torch.randn(x.shape, generator=g, device=DEV).to(dtype) for x in (q, k)]
    w = (1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    tables = [t.to(DEV) for t in _tables(T, rot)]
    lens = _i32([T, T - T // 3]).to(DEV)
    out = qk_norm_rope(q, k, *tables, w, w, lens=lens, interleaved=interleaved)
    grads = torch.autograd.grad(out, (q, k), up)
    for t0 in range(0, T, -(-T // 5)):
        t1 = min(T, t0 + -(-T // 5))
        part = [x.detach()[:, :, t0:t1].requires_grad_() for x in (q, k)]
        at = torch.arange(t0, t1, dtype=torch.int32, device=DEV).expand(B, -1)
        got = qk_norm_rope(*part, *tables, w, w, lens=(lens - t0).clamp(min=0).int(), positions=at, interleaved=interleaved)
        for a, b in zip(got, out):
            assert torch.equal(a, b[:, :, t0:t1])
        for a, b in zip(torch.autograd.grad(got, part, [x[:, :, t0:t1] for x in up]), grads):
            assert torch.equal(a, b[:, :, t0:t1])


def test_more_than_two_to_the_31_elements():
    g = torch.Generator(device=DEV).manual_seed(11)
    B, Hq, Hkv, T, D = 4, 40, 2, 110000, 128
    assert B * Hq * T * D > 1 << 31
    q, k, gq, gk = (torch.randn(B, h, T, D, generator=g, device=DEV, dtype=torch.bfloat16) for h in (Hq, Hkv, Hq, Hkv))
    tables = _tables(T, D)
    q.requires_grad_(), k.requires_grad_()
    out = qk_norm_rope(q, k, *[t.to(DEV) for t in tables])
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for b, h, t in ((0, 0, slice(0, 50)), (B - 1, Hq - 1, slice(T - 50, T)), (2, 17, slice(70000, 70050))):
        want = kv_oracle.rope_rows(q[b, h, t].detach().cpu(), tables[0][t], tables[1][t], None, 1e-6, False, gq[b, h, t].cpu())
        kv_oracle.assert_within("out", out[0][b, h, t], want["out"])
        kv_oracle.assert_within("dx", grads[0][b, h, t], want["dx"])
