"""The MXFP4 and windowed-attention operators as a model uses them: together in
a block, behind the row shims, captured into graphs, on side streams, with
weights and inputs that change right before a call."""
import pytest
import torch
from torch import nn

from h3_engine_b200 import mxfp4, ops
from h3_engine_b200.blocks import AttnBlock, window_pairs
from tests import mx_ref as ref
from tests.test_attention_window import attend, check_packed, seen_mask
from tests.test_mxfp4 import BF16, F16, rand


# ---------------------------------------------------------------- CPU
@pytest.mark.parametrize("rule", [(None, None, 0, False), (3, 2, 0, False), (0, 0, 4, False),
                                  (5, 0, 3, True), (None, 0, 0, True), (2, None, 9, False)])
@pytest.mark.parametrize("n", [0, 1, 4, 20])
def test_window_pairs_counts_what_is_seen(rule, n):
    assert window_pairs(n, rule[:2], *rule[2:]) == int(seen_mask(n, n, *rule).sum())
    assert window_pairs(n, None) == n * n


def test_windowed_block_refusals():
    w = torch.zeros(1)
    with pytest.raises(ValueError):
        AttnBlock(w, w, w, w, w, None, None, 1, sinks=2)
    with pytest.raises(ValueError):
        AttnBlock(w, w, w, w, w, None, None, 1, causal=True)


def test_shims_leave_what_mxfp4_does_not_take():
    from h3_engine_b200.kernels import ffn_qkvo_gemms as gm
    lin = nn.Linear(64, 64, bias=False)
    x = torch.zeros(2, 64)
    assert gm.qkv_kernel(lin, lin, lin, x) is gm.MISS
    assert gm.out_kernel(lin, x) is gm.MISS
    assert mxfp4.shared_qkv(lin, lin, lin, x) is None


# ---------------------------------------------------------------- GPU: a block

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_projections_attention_and_feed_forward_together(cuda, dtype):
    """x + Wo attention(Wq x, Wk x, Wv x), then + the gated feed-forward: every
    stage against 64 bits on the values that the stage before gave."""
    docs, heads, kv, d, f = [130, 1, 0, 70], 4, 2, 64, 256
    t, c = sum(docs), 4 * 64
    cu = [0, 130, 131, 131, 201]
    rule = (40, 0, 3, True)
    x = rand(t, c, seed=1).to(dtype)
    lin = {n: nn.Linear(c, o, bias=False).requires_grad_(False) for n, o in
           (("q", heads * d), ("k", kv * d), ("v", kv * d), ("o", c), ("up", 2 * f))}
    lin["down"] = nn.Linear(f, c, bias=False).requires_grad_(False)
    for i, m in enumerate(lin.values()):
        m.weight.data = rand(*m.weight.shape, seed=20 + i, scale=m.in_features ** -0.5).to(BF16)
    mods = {n: mxfp4.MXFP4Linear(m.to(cuda)) for n, m in lin.items()}
    xg = x.to(cuda)
    q, k, v = mxfp4.shared_qkv(mods["q"], mods["k"], mods["v"], xg)
    for got, n in ((q, "q"), (k, "k"), (v, "v")):
        assert torch.equal(got, mods[n](xg))                     # fused or apart, the same
    o = ops.attention_window(q, k, v, heads, d, cu, kv_heads=kv, window=rule[:2], sinks=rule[2],
                             causal=rule[3])
    check_packed(o.cpu(), q.cpu(), k.cpu(), v.cpu(), cu, cu, heads, kv, d, rule)
    h = mxfp4.mxfp4_linear(mods["o"].weight_mxfp4, o, residual=xg)
    y, dy = ref.product(ref.quantize(o)[0], ref.quantize(lin["o"].weight)[0])
    want = y + x.double()
    half = ref.half_step(dtype)
    off = dy + 2.0 ** -23 * want.abs()
    assert ((h.cpu().double() - want).abs() <= off + half * (want.abs() + off) + 1e-7).all()
    z = mxfp4.linear_ffn(mods["up"], mods["down"], h)
    up = mxfp4.gated_up_weight(lin["up"].weight.to(cuda))
    assert torch.equal(z, mxfp4.gated_ffn(up, mods["down"].weight_mxfp4, h))
    # the feed-forward may write over its input, which is its residual too
    s = h.clone()
    mxfp4.gated_ffn(up, mods["down"].weight_mxfp4, s, residual=s, out=s)
    assert ((s.double() - (h.double() + z.double())).abs()
            <= 2 * half * (h.double().abs() + 2 * z.double().abs()) + 1e-7).all()


@pytest.mark.gpu
def test_row_shims_take_mxfp4_linears(cuda, monkeypatch):
    from h3_engine_b200.kernels import ffn_qkvo_gemms as gm
    monkeypatch.setenv("H3_NVFP4", "1")

    class Gate(nn.Module):
        def __init__(self, proj):
            super().__init__()
            self.proj, self.activation = proj, nn.SiLU()

        def forward(self, x):
            value, gate = self.proj(x).chunk(2, -1)
            return value * self.activation(gate)

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            def lin(k, n):
                return nn.Linear(k, n, bias=False)
            self.attn = nn.Module()
            self.attn.to_q, self.attn.to_k, self.attn.to_v = lin(128, 128), lin(128, 128), lin(128, 128)
            self.attn.to_out = nn.ModuleList([lin(128, 128), nn.Identity()])
            self.ff = nn.Module()
            self.ff.net = nn.ModuleList([Gate(lin(128, 512)), nn.Identity(), lin(256, 128)])

    torch.manual_seed(0)
    model = nn.Module()
    model.transformer_blocks = nn.ModuleList([Block()]).to(cuda).to(BF16).requires_grad_(False)
    assert mxfp4.quantize_blocks(model) == {"linears_quantized": 6}
    b = model.transformer_blocks[0]
    x = rand(2, 33, 128, seed=4).to(BF16).to(cuda)
    a = b.attn
    for got, m in zip(gm.qkv_projection(a.to_q, a.to_k, a.to_v, x), (a.to_q, a.to_k, a.to_v)):
        assert torch.equal(got, m(x))
    assert torch.equal(gm.out_projection(a.to_out[0], x), a.to_out[0](x))
    y = gm.ffn(b.ff, x)
    assert y.shape == x.shape
    up = mxfp4.MXFP4Weight.from_packed(b.ff.net[0].proj.weight_mxfp4.qdata,
                                       b.ff.net[0].proj.weight_mxfp4.scale, 512, 128)
    deq = up.dequantize(torch.float32)
    again = mxfp4.gated_ffn(mxfp4.gated_up_weight(deq), b.ff.net[2].weight_mxfp4, x)
    assert torch.equal(y, again)          # quantizing MXFP4 values gives them back


@pytest.mark.gpu
def test_windowed_attention_block(cuda):
    """AttnBlock with a window: its attention is ``attention_window`` of its own
    q, k and v; a window over everything gives the block without one."""
    t, c, heads = 300, 256, 2
    cu = [0, 200, 300]
    w = [rand(c, c, seed=30 + i, scale=c ** -0.5).to(BF16).to(cuda) for i in range(4)]
    gamma = torch.ones(c, dtype=BF16, device=cuda)
    x = rand(t, c, seed=5).to(BF16).to(cuda)
    block = AttnBlock(*w, gamma, None, None, heads, window=(50, 20), sinks=4)
    block(x, None, cu)
    ws = next(v for k, v in block._ws.items() if k[0] == "attn")
    qkv, o = ws["qkv"].cpu(), ws["o"].cpu()
    check_packed(o, *qkv.split(c, 1), cu, cu, heads, heads, 128, (50, 20, 4, False))
    assert block.flops(t, cu)["attention"] == 4 * c * sum(
        int(seen_mask(n, n, 50, 20, 4, False).sum()) for n in (200, 100))
    full = AttnBlock(*w, gamma, None, None, heads)
    wide = AttnBlock(*w, gamma, None, None, heads, window=(None, None))
    full(x, None, cu)
    wide(x, None, cu)
    pick = lambda b: next(v for k, v in b._ws.items() if k[0] == "attn")["o"].cpu().double()  # noqa: E731
    for s, e in zip(cu, cu[1:]):
        for h in range(heads):
            q, k, v = (z[s:e, h * 128:h * 128 + 128] for z in qkv.split(c, 1))
            _, off = attend(q, k, v, seen_mask(e - s, e - s, None, None, 0, False), 128 ** -0.5,
                            2.0 ** -8)
            a, b = (pick(m)[s:e, h * 128:h * 128 + 128] for m in (full, wide))
            assert ((a - b).abs() <= 2 * off).all()


# ---------------------------------------------------------------- GPU: streams and graphs
def _calls(cuda, m):
    """(name, function of one input, input shape, type) of every operator at m rows."""
    k, n, f = 288, 136, 384
    w = mxfp4.MXFP4Weight(rand(n, k, seed=1, scale=k ** -0.5).to(BF16).to(cuda))
    up = mxfp4.gated_up_weight(rand(2 * f, k, seed=2, scale=k ** -0.5).to(BF16).to(cuda))
    down = mxfp4.MXFP4Weight(rand(k, f, seed=3, scale=f ** -0.5).to(BF16).to(cuda))

    def quant(x):
        return ops.mxfp4_dequantize(*ops.mxfp4_quantize(x), x.shape[0], k)

    def window(x):
        q, kk, v = x[:, :128], x[:, 128:192], x[:, 192:256]
        return ops.attention_window(q, kk, v, 2, 64, [0, m // 3, m], kv_heads=1, window=(30, 10),
                                    sinks=2)

    return [("quantize", quant), ("linear", lambda x: mxfp4.mxfp4_linear(w, x, act="gelu")),
            ("ffn", lambda x: mxfp4.gated_ffn(up, down, x, residual=x)), ("window", window)], k


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_graph_replays_follow_their_inputs(cuda, m):
    """Two graphs per operator, replayed in turn and mixed with eager calls."""
    calls, k = _calls(cuda, m)
    inputs = [rand(m, k, seed=50 + i).to(BF16).to(cuda) for i in range(4)]
    for name, fn in calls:
        want = [fn(x).clone() for x in inputs]
        graphs = []
        for _ in range(2):
            x = inputs[0].clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                fn(x)
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = fn(x)
            graphs.append((g, x, y))
        for i in range(6):
            g, x, y = graphs[i % 2]
            x.copy_(inputs[i % 4])
            g.replay()
            got = y.clone()
            assert torch.equal(fn(inputs[(i + 1) % 4]), want[(i + 1) % 4]), name
            assert torch.equal(got, want[i % 4]), name


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 40, 300])
def test_two_streams_at_once(cuda, m):
    calls, k = _calls(cuda, m)
    inputs = [rand(m, k, seed=60 + i).to(BF16).to(cuda) for i in range(2)]
    for name, fn in calls:
        want = [fn(x).clone() for x in inputs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in inputs]
        got = [[], []]
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(fn(inputs[i]))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(y, want[i]) for y in got[i]), name


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 9, 64, 200])
def test_weights_and_inputs_written_just_before(cuda, m):
    """A weight that the same stream quantized into the same buffers a moment
    ago, an input that a kernel is still writing when the call is made."""
    n, k, f = 256, 512, 256
    ws = [rand(n, k, seed=70 + i, scale=k ** -0.5).to(BF16).to(cuda) for i in range(4)]
    xs = [rand(m, k, seed=80 + i).to(BF16).to(cuda) for i in range(4)]
    want = []
    for w, x in zip(ws, xs):
        want.append(mxfp4.mxfp4_linear(mxfp4.MXFP4Weight(w), x))
        torch.cuda.synchronize()
    q, sf = ops.mxfp4_quantize(ws[0])
    x = torch.empty_like(xs[0])
    got = []
    for i in range(40):
        ops.mxfp4_quantize(ws[i % 4], q_out=q, sf_out=sf)
        x.copy_(xs[i % 4])
        got.append(ops.mxfp4_linear(x, q, sf, n, k))
        qa, sfa = ops.mxfp4_quantize(x)
        got.append(ops.mxfp4_gemm(qa, sfa, m, q, sf, n, k))
    for i in range(40):
        assert torch.equal(got[2 * i], want[i % 4]) and torch.equal(got[2 * i + 1], want[i % 4])
    downs = [rand(k, f, seed=90 + i, scale=f ** -0.5).to(BF16).to(cuda) for i in range(4)]
    up = mxfp4.gated_up_weight(rand(2 * f, k, seed=99, scale=k ** -0.5).to(BF16).to(cuda))
    want = []
    for w, y in zip(downs, xs):
        want.append(mxfp4.gated_ffn(up, mxfp4.MXFP4Weight(w), y))
        torch.cuda.synchronize()
    q, sf = ops.mxfp4_quantize(downs[0])
    down = mxfp4.MXFP4Weight.from_packed(q, sf, k, f)
    got = []
    for i in range(40):
        ops.mxfp4_quantize(downs[i % 4], q_out=q, sf_out=sf)
        x.copy_(xs[i % 4])
        got.append(mxfp4.gated_ffn(up, down, x))
    for i in range(40):
        assert torch.equal(got[i], want[i % 4])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 12, 100, 300])
def test_calls_in_a_row_follow_each_other(cuda, m):
    """Kernels come up under the end of the one before: in a row without a pause,
    eager and captured, calls that reuse one another's buffers give what they
    give with a synchronisation after each."""
    d, f = 256, 512
    w = mxfp4.MXFP4Weight(rand(d, d, scale=0.1).to(BF16).to(cuda))
    up = mxfp4.gated_up_weight(rand(2 * f, d, seed=1, scale=0.1).to(BF16).to(cuda))
    down = mxfp4.MXFP4Weight(rand(d, f, seed=2, scale=0.1).to(BF16).to(cuda))
    x0 = rand(m, d, seed=3).to(BF16).to(cuda)
    cache = rand(2, 600, 2, 128, seed=4).to(BF16).to(cuda)
    n = torch.tensor([m + 300, 7], dtype=torch.int32, device=cuda)
    a, b, o = (torch.empty_like(x0) for _ in range(3))
    q, sf = ops.mxfp4_quantize(x0)
    x, dec = x0.clone(), torch.empty(2, 1, 2, 128, dtype=BF16, device=cuda)

    def step(pause):
        mxfp4.mxfp4_linear(w, x, residual=x0, out=a)
        pause()
        ops.attention_window(a, x, x0, 2, 128, [0, m], window=(40, 40), sinks=2, out=o)
        pause()
        cache[0, :1].copy_(o.view(m, 2, 128)[:1])
        pause()
        ops.attention_window_decode(o[-1:].view(1, 1, 2, 128).expand(2, 1, 2, 128), cache, cache, n,
                                    out=dec)
        pause()
        o[:1] += dec[0].view(1, d)
        pause()
        mxfp4.gated_ffn(up, down, o, residual=a, out=b)
        pause()
        ops.mxfp4_quantize(b, q_out=q, sf_out=sf)
        pause()
        ops.mxfp4_dequantize(q, sf, m, d, out=x)
        pause()
        ops.mxfp4_gemm(q, sf, m, w.qdata, w.scale, d, d, residual=x, out=x)
        pause()
        torch.clamp_(x, -4, 4)
        pause()

    def reset():
        x.copy_(x0)
        cache[0, :1].zero_()

    reset()
    for _ in range(6):
        step(torch.cuda.synchronize)
    want = x.clone(), dec.clone()
    for _ in range(10):
        reset()
        for _ in range(6):
            step(lambda: None)
        assert torch.equal(x, want[0]) and torch.equal(dec, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            for _ in range(6):
                step(lambda: None)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(10):
        reset()
        graph.replay()
        assert torch.equal(x, want[0]) and torch.equal(dec, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 700])
def test_streams_that_fork_and_join(cuda, m):
    """A kernel with two predecessors, on its own stream and on another, eager
    and captured: it follows both, and what they read is not written before."""
    d, f = 256, 512
    w = mxfp4.MXFP4Weight(rand(d, d, scale=0.1).to(BF16).to(cuda))
    up = mxfp4.gated_up_weight(rand(2 * f, d, seed=1, scale=0.1).to(BF16).to(cuda))
    down = mxfp4.MXFP4Weight(rand(d, f, seed=2, scale=0.1).to(BF16).to(cuda))
    x0 = rand(m, d, seed=3).to(BF16).to(cuda)
    x, a, b, h, o = (torch.empty_like(x0) for _ in range(5))
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            mxfp4.gated_ffn(up, down, x, out=h)
            mxfp4.mxfp4_linear(w, h, residual=x, out=b)
        mxfp4.mxfp4_linear(w, x, act="gelu", out=a)
        main.wait_stream(side)
        ops.attention_window(a, b, x, 2, 128, [0, m], window=(600, 5), sinks=1, out=o)
        mxfp4.mxfp4_linear(w, o, residual=b, out=x)

    def alone():
        mxfp4.gated_ffn(up, down, x, out=h)
        torch.cuda.synchronize()
        mxfp4.mxfp4_linear(w, h, residual=x, out=b)
        torch.cuda.synchronize()
        mxfp4.mxfp4_linear(w, x, act="gelu", out=a)
        torch.cuda.synchronize()
        ops.attention_window(a, b, x, 2, 128, [0, m], window=(600, 5), sinks=1, out=o)
        torch.cuda.synchronize()
        mxfp4.mxfp4_linear(w, o, residual=b, out=x)
        torch.cuda.synchronize()

    x.copy_(x0)
    for _ in range(4):
        alone()
    want = x.view(torch.int16).clone()       # bits: the values grow from step to step
    for _ in range(10):
        x.copy_(x0)
        for _ in range(4):
            step()
        assert torch.equal(x.view(torch.int16), want)
    capture = torch.cuda.Stream()
    capture.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(capture):
        with torch.cuda.graph(graph, stream=capture):
            for _ in range(4):
                step()
    torch.cuda.current_stream().wait_stream(capture)
    for _ in range(10):
        x.copy_(x0)
        graph.replay()
        assert torch.equal(x.view(torch.int16), want)


@pytest.mark.gpu
def test_outputs_must_stand_apart(cuda):
    w = mxfp4.MXFP4Weight(rand(64, 64).to(BF16).to(cuda))
    buf = rand(9, 64).to(BF16).to(cuda)
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, buf[:8], out=buf[:8])
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, rand(8, 64).to(BF16).to(cuda), residual=buf[:8], out=buf[1:])
    r = buf[:8].clone()
    x = rand(8, 64, seed=2).to(BF16).to(cuda)
    want = mxfp4.mxfp4_linear(w, x, residual=r)
    assert torch.equal(mxfp4.mxfp4_linear(w, x, residual=r, out=r), want)
    q, sf = ops.mxfp4_quantize(x)
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x, q_out=q, sf_out=q.view(-1))
    kv = rand(8, 128, seed=3).to(BF16).to(cuda)
    with pytest.raises(ValueError):
        ops.attention_window(kv.clone(), kv, kv, 1, 128, [0, 8], out=kv)
    qq = kv.clone()
    want = ops.attention_window(qq, kv, kv, 1, 128, [0, 8], window=(2, 2))
    assert torch.equal(ops.attention_window(qq, kv, kv, 1, 128, [0, 8], window=(2, 2), out=qq), want)
    c = rand(1, 8, 1, 128, seed=4).to(BF16).to(cuda)
    n = torch.tensor([8], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        ops.attention_window_decode(c[:, :1].clone(), c, c, n, out=c[:, :1])


@pytest.mark.gpu
def test_outputs_in_rows_that_hold_other_columns(cuda):
    """Columns beside the inputs' in the same rows are free; columns that reach
    into an input's are refused, whatever the layout."""
    d = 64
    buf = rand(40, 6 * d).to(BF16).to(cuda)
    q, k, v = buf[:, :d], buf[:, d:2 * d], buf[:, 2 * d:3 * d]
    args = (1, d, [0, 40])
    want = ops.attention_window(q, k, v, *args, window=(3, 3))
    got = ops.attention_window(q, k, v, *args, window=(3, 3), out=buf[:, 3 * d:4 * d])
    assert torch.equal(got, want)
    for bad in (buf[:, d:2 * d], buf[:, d // 2:d // 2 + d], buf[:, 2 * d + 8:3 * d + 8]):
        with pytest.raises(ValueError):
            ops.attention_window(q, k, v, *args, out=bad)
    assert torch.equal(ops.attention_window(q, k, v, *args, window=(3, 3), out=q), want)

    w = mxfp4.MXFP4Weight(rand(d, 2 * d, seed=1, scale=0.1).to(BF16).to(cuda))
    x = buf[:, 4 * d:]
    r3 = buf[:, :d].unflatten(0, (4, 10))            # the same rows, one more dimension
    want = mxfp4.mxfp4_linear(w, x, residual=r3)
    assert torch.equal(mxfp4.mxfp4_linear(w, x, residual=r3, out=buf[:, 3 * d:4 * d]), want)
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, out=buf[:, 5 * d:])
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, residual=r3, out=buf[:, 8:8 + d])
    rows = buf[:20, :d]
    with pytest.raises(ValueError):                  # the same columns, two rows on
        mxfp4.mxfp4_linear(w, x[:20], residual=rows, out=buf[2:22, :d])
    assert torch.equal(mxfp4.mxfp4_linear(w, x, residual=r3, out=buf[:, :d]), want)


@pytest.mark.gpu
def test_results_carry_no_gradient(cuda):
    x = rand(20, 128).to(BF16).to(cuda).requires_grad_()
    w = mxfp4.MXFP4Weight(rand(64, 128, scale=0.1).to(BF16).to(cuda))
    y = mxfp4.mxfp4_linear(w, x)
    a = ops.attention_window(x, x, x, 1, 128, [0, 20])
    c = x.view(1, 20, 1, 128)
    d = ops.attention_window_decode(c[:, -1:], c, c, torch.tensor([20], dtype=torch.int32).to(cuda))
    for t in (y, a, d):
        assert not t.requires_grad and t.grad_fn is None
    with pytest.raises(RuntimeError):
        (y.float().sum() + a.float().sum()).backward()


@pytest.mark.gpu
def test_compiled_callers_keep_the_operators(cuda):
    w = mxfp4.MXFP4Weight(rand(64, 128, scale=0.1).to(BF16).to(cuda))
    x = rand(20, 128).to(BF16).to(cuda)

    def step(x):
        y = mxfp4.mxfp4_linear(w, x, act="gelu")
        return ops.attention_window(y, y, y, 1, 64, [0, 20], window=(4, 4), sinks=1) + 1

    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x)
    assert torch.equal(got, step(x))
