"""Windowed attention whose items are cut along their keys (counters and partial
results in a workspace): captured, replayed, on two streams, in a row."""
import ctypes

import pytest
import torch

from h3_engine_b200 import _lib, mxfp4, ops
from tests.test_attention_window import BF16, F16, check_packed, packed_case

CASES = {        # query and key lengths, heads, key heads, head_dim, type, rule
    "items of 128": ([1500], [1500], 2, 2, 128, BF16, (None, None, 0, False)),
    "items of 256": ([2100], [2100], 8, 4, 128, F16, (None, None, 3, True)),
    "head_dim 64": ([2200], [2200], 2, 1, 64, BF16, (1400, 300, 70, False)),
    "two launches": ([3 + i % 4 for i in range(70)], [1100 + 3 * i for i in range(70)], 1, 1, 64,
                     F16, (None, None, 0, True)),
}


def workspace(lq, lk, heads, d, rule):
    arr = [(ctypes.c_int32 * len(t))(*t) for t in (lq, lk)]
    left, right = ((1 << 30) - 1 if s is None else s for s in rule[:2])
    return _lib.lib().h3b_attention_window_ws(*arr, len(lq), heads, d, left, right, rule[2])


def case(name, cuda, inputs=4):
    lq, lk, heads, kv, d, dtype, rule = CASES[name]
    assert workspace(lq, lk, heads, d, rule) > 0
    host = [packed_case(lq, lk, heads, kv, d, dtype, seed=20 + i) for i in range(inputs)]
    cq, ck = host[0][3:]

    def call(x, out=None):
        return ops.attention_window(*x, heads, d, cq, kv_heads=kv, cu_seqlens_k=ck,
                                    window=rule[:2], sinks=rule[2], causal=rule[3], out=out)

    dev = [[t.to(cuda) for t in h[:3]] for h in host]
    want = []
    for x, h in zip(dev, host):
        want.append(call(x))
        torch.cuda.synchronize()
    check_packed(want[0].cpu(), *host[0], heads, kv, d, rule)
    return call, dev, want


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_graphs_follow_their_inputs(cuda, name):
    """Two graphs, replayed in turn and mixed with eager calls."""
    call, inputs, want = case(name, cuda)
    graphs = []
    for _ in range(2):
        x = [t.clone() for t in inputs[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                y = call(x)
                z = call(x)              # the same memory again, perhaps
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((g, x, y, z))
    for i in range(8):
        g, x, y, z = graphs[i % 2]
        for t, s in zip(x, inputs[i % 4]):
            t.copy_(s)
        g.replay()
        got = y.clone(), z.clone()
        assert torch.equal(call(inputs[(i + 1) % 4]), want[(i + 1) % 4])
        assert torch.equal(got[0], want[i % 4]) and torch.equal(got[1], want[i % 4])


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("captured", [False, True])
def test_two_streams_at_once(cuda, name, captured):
    call, inputs, want = case(name, cuda, 2)
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    graphs = []
    for s, x in zip(streams, inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            with torch.cuda.graph(g, stream=s):
                y = call(x)
        graphs.append((g, y))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if captured:
                    graphs[i][0].replay()
                    got[i].append(graphs[i][1].clone())
                else:
                    got[i].append(call(inputs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_calls_in_a_row(cuda, d):
    """Each call reads what the one before wrote, whole and split items and other
    operators in turn; eager and captured as with a synchronisation after each."""
    t, heads = 1500, 2
    c = heads * d
    rules = [((None, None), 0, False), ((200, 30), 4, True), ((1000, 0), 900, False)]
    assert any(workspace([t], [t], heads, d, (*w, s, k)) > 0 for w, s, k in rules)
    assert workspace([t], [t], heads, d, (None, None, 0, False)) > 0
    w = mxfp4.MXFP4Weight(torch.randn(c, c, generator=torch.Generator().manual_seed(1))
                          .mul(c ** -0.5).to(BF16).to(cuda))
    x0 = torch.randn(t, c, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    x, a, o = (torch.empty_like(x0) for _ in range(3))

    def step(pause):
        for window, sinks, causal in rules:
            mxfp4.mxfp4_linear(w, x, residual=x0, out=a)
            pause()
            ops.attention_window(x, a, x, heads, d, [0, t], window=window, sinks=sinks,
                                 causal=causal, out=o)
            pause()
            ops.attention_window(o, a, x0, heads, d, [0, t], window=window, sinks=sinks,
                                 causal=causal, out=o)
            pause()
            mxfp4.mxfp4_linear(w, o, residual=a, out=x)
            pause()
            torch.clamp_(x, -4, 4)
            pause()

    def run(pause, steps=3):
        x.copy_(x0)
        for _ in range(steps):
            step(pause)

    run(torch.cuda.synchronize)
    want = x.clone()
    for _ in range(6):
        run(lambda: None)
        assert torch.equal(x, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run(lambda: None)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(6):
        graph.replay()
        assert torch.equal(x, want)


# ---------------------------------------------------------------- documents of uneven lengths
def test_a_short_document_leaves_the_others_their_parts():
    """The workspace of one long history is not lost to a short document beside it."""
    rule = (None, None, 0, True)
    alone = workspace([16], [16000], 1, 128, rule)
    assert alone > 0
    for lq, lk in (([16, 1], [16000, 1]), ([1, 16], [1, 16000]), ([16, 5], [16000, 0]),
                   ([16, 0], [16000, 0]), ([16, 3, 8], [16000, 700, 8])):
        assert workspace(lq, lk, 1, 128, rule) >= alone


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("rule", [(None, None, 0, True), (None, None, 0, False), (3000, 0, 5, True),
                                  (40, 30, 300, False)])
def test_parts_of_uneven_documents(cuda, heads, kv, d, dtype, rule):
    """One long history beside documents that fill some of its parts, one or none."""
    lq = [16, 1, 5, 300, 7, 130, 0, 40]
    lk = [9000, 1, 0, 700, 3000, 60, 50, 1100]
    q, k, v, cq, ck = packed_case(lq, lk, heads, kv, d, dtype, seed=30)
    if rule[0] != 40:
        assert workspace(lq, lk, heads, d, rule) > 0
    args = [t.to(cuda) for t in (q, k, v)]

    def call():
        return ops.attention_window(*args, heads, d, cq, kv_heads=kv, cu_seqlens_k=ck,
                                    window=rule[:2], sinks=rule[2], causal=rule[3])

    got = call()
    check_packed(got.cpu(), q, k, v, cq, ck, heads, kv, d, rule)
    for _ in range(5):                   # whichever part is last, and counters left at 0
        assert torch.equal(call(), got)
