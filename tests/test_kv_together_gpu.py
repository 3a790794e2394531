"""Cross attention, attention over pages and appending as a program uses them together: captured, on several streams and host
threads at once, on shared pages, and past 2^31 elements."""
import threading

import pytest
import torch

from cross_attention import cross_attention
from oracle import kv_oracle
from paged_attention import paged_append, paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (type, B, Hq, Hkv, Tq, Tk, D, lens): tile kernels divided and whole, the wide ones, the hand-scheduled ones, one token
SHAPES = [
    (torch.float32, 2, 4, 4, 60, 700, 64, [700, 33]),
    (torch.float32, 2, 4, 2, 70, 200, 256, [200, 7]),
    (torch.float16, 8, 16, 16, 260, 300, 64, None),
    (torch.bfloat16, 4, 8, 8, 333, 900, 256, [900, 1, 450, 0]),
    (torch.bfloat16, 3, 6, 2, 200, 300, 256, [300, 299, 64]),
    (torch.bfloat16, 8, 16, 16, 500, 600, 128, [600, 0, 64, 65, 599, 300, 31, 512]),
    (torch.float16, 4, 32, 8, 512, 700, 128, None),
    (torch.bfloat16, 4, 8, 2, 1, 4000, 128, [4000, 1, 0, 2222]),
]


def _tensors(shape, seed):
    dtype, B, Hq, Hkv, Tq, Tk, D, _ = shape
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((B, Hq, Tq, D), (B, Hkv, Tk, D), (B, Hkv, Tk, D), (B, Hq, Tq, D))]


def _lens(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def _step(x, lens):
    leaves = [t.detach().requires_grad_() for t in x[:3]]
    o = cross_attention(*leaves, lens)
    return (o.detach(), *torch.autograd.grad(o, leaves, x[3]))


@pytest.mark.parametrize("shape", SHAPES)
def test_two_graphs(shape):
    """Two captures of forward and backward, replayed in turn, on two streams at once and with eager calls between."""
    lens = _lens(shape[-1])
    static = [_tensors(shape, s) for s in (1, 2)]
    fresh = [_tensors(shape, s) for s in (3, 4)]
    _step(static[0], lens)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(x, lens))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for values in (static, fresh, fresh):
        values = [[t.clone() for t in x] for x in values]
        want = [_step(x, lens) for x in values]
        for s, x in zip(static, values):
            for a, b in zip(s, x):
                a.copy_(b)
        for graph, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b)
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b)


def test_host_threads():
    """Calls from several threads, each on a stream of its own."""
    work = [(s, _tensors(s, i), _lens(s[-1])) for i, s in enumerate(SHAPES)]
    want = [_step(x, lens) for _, x, lens in work]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = _step(work[i][1], work[i][2])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(work[i][0])

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype,B,Hq,Hkv,Tq,Tk,D", [(torch.bfloat16, 64, 64, 64, 4100, 512, 128), (torch.float16, 64, 64, 16, 8200, 40, 64)])
def test_more_than_two_to_the_31_elements(dtype, B, Hq, Hkv, Tq, Tk, D):
    assert B * Hq * Tq * D > 1 << 31
    g = torch.Generator(device=DEV).manual_seed(11)
    q, k, v, d_o = (torch.randn(*s, generator=g, device=DEV, dtype=dtype) for s in ((B, Hq, Tq, D), (B, Hkv, Tk, D), (B, Hkv, Tk, D), (B, Hq, Tq, D)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = cross_attention(*leaves, return_lse=True)
    grads = torch.autograd.grad(o, leaves, d_o)
    G = Hq // Hkv
    for b, h in ((0, 0), (B - 1, Hkv - 1)):
        heads = slice(h * G, (h + 1) * G)
        one = [t[b:b + 1].detach().cpu() for t in (q[:, heads], k[:, h:h + 1], v[:, h:h + 1], d_o[:, heads])]
        want = kv_oracle.cross(*one[:3], None, None, None, one[3])
        for name, got in (("o", o[b:b + 1, heads]), ("lse", lse[b:b + 1, heads]), ("dq", grads[0][b:b + 1, heads]),
                          ("dk", grads[1][b:b + 1, h:h + 1]), ("dv", grads[2][b:b + 1, h:h + 1])):
            kv_oracle.assert_within(f"{name} of {b}", got, want[name])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_sequences_that_share_pages(dtype):
    """A common prefix stands in the cache once."""
    B, Hq, Hkv, D, page, prefix = 5, 8, 2, 64, 16, 640
    lens = [641, 700, 656, 900, 640]
    g = torch.Generator().manual_seed(8)
    width, shared = 60, prefix // page
    own = torch.arange(B * (width - shared), dtype=torch.int32).view(B, -1) + shared
    table = torch.cat([torch.arange(shared, dtype=torch.int32).expand(B, -1), own], 1)
    k, v = (torch.randn(int(table.max()) + 1, Hkv, page, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(B, Hq, 1, D, generator=g).to(dtype).to(DEV)
    apart = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    got = paged_attention(q, k, v, table.to(DEV), _lens(lens))
    want = paged_attention(q, k[table.long().to(DEV).flatten()], v[table.long().to(DEV).flatten()], apart, _lens(lens))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decoder_layer_in_chunks(dtype):
    """A decoder's attention, chunk by chunk: appending, over the cache in pages, and then over an encoder's states."""
    B, Hq, Hkv, D, page, C, R, T, Tk = 3, 8, 4, 64, 16, 12, 3, 96, 150
    g = torch.Generator().manual_seed(9)
    q, k, v, states_k, states_v = (torch.randn(B, h, t, D, generator=g).to(dtype).to(DEV)
                                   for h, t in ((Hq, T), (Hkv, T), (Hkv, T), (Hkv, Tk), (Hkv, Tk)))
    state_lens = _lens([150, 1, 77])
    width = T // page
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).to(DEV)
    k_pages, v_pages = (torch.full((B * width, Hkv, page, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    rows, crossed = [], []
    with torch.no_grad():
        for t in range(0, T, C):
            lens = torch.full((B,), t + C, dtype=torch.int32, device=DEV)
            paged_append(k[:, :, t:t + C], v[:, :, t:t + C], k_pages, v_pages, table, lens)
            rows.append(paged_attention(q[:, :, t:t + C], k_pages, v_pages, table, lens, C, R))
            crossed.append(cross_attention(rows[-1], states_k, states_v, state_lens))
        rows, crossed = torch.cat(rows, 2), torch.cat(crossed, 2)
        for b in range(0, T, C):   # each chunk, as it stood in the cache when it was the newest
            lens = torch.full((B,), b + C, dtype=torch.int32)
            want = kv_oracle.paged(q[:, :, b:b + C].cpu(), k_pages.cpu(), v_pages.cpu(), table.cpu(), lens, C, R, None, None)
            kv_oracle.assert_within("o", rows[:, :, b:b + C], want["o"])
        want = kv_oracle.cross(rows.cpu(), states_k.cpu(), states_v.cpu(), state_lens.cpu())
        kv_oracle.assert_within("o", crossed, want["o"])
