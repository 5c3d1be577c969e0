"""Weights that change under MXFP4 modules: the fused q | k | v weight and the
reordered up projection, which are copies, follow the weights they were made of."""
import copy

import pytest
import torch
from torch import nn

from h3_engine_b200 import mxfp4, ops
from h3_engine_b200.kernels import ffn_qkvo_gemms as gm
from h3_engine_b200.nvfp4 import _unswizzle

K, F = 128, 256


def lin(n, k, seed, device="cpu"):
    m = nn.Linear(k, n, bias=False).requires_grad_(False)
    g = torch.Generator().manual_seed(seed)
    m.weight.data = (torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16)
    return mxfp4.MXFP4Linear(m.to(device))


class Gate(nn.Module):
    def __init__(self, proj):
        super().__init__()
        self.proj, self.activation = proj, nn.SiLU()


class FeedForward(nn.Module):
    def __init__(self, up, down):
        super().__init__()
        self.net = nn.ModuleList([Gate(up), nn.Identity(), down])


def modules(device="cpu"):
    return ([lin(n, K, 1 + i, device) for i, n in enumerate((256, 128, 128))],
            lin(2 * F, K, 5, device), lin(K, F, 6, device))


def rewrite(w, seed, device="cpu"):
    """Other codes and scales into the weight's own tensors, as a call writes them."""
    other = lin(w.out_features, w.in_features, seed, device).weight_mxfp4
    w.qdata.copy_(other.qdata)
    w.scale.copy_(other.scale)


def rebind(w, seed, device="cpu"):
    other = lin(w.out_features, w.in_features, seed, device).weight_mxfp4
    w.qdata, w.scale = other.qdata, other.scale


def replace(m, seed, device="cpu"):
    m.weight_mxfp4 = lin(m.out_features, m.in_features, seed, device).weight_mxfp4


@pytest.fixture
def on_cpu(monkeypatch):
    """The operators as sums over the bytes of codes and scales, on the CPU."""
    def quantize(x, **_):
        q = (x.float()[:, ::2] * 977 + x.float()[:, 1::2] * 31).mul(7).to(torch.int64) % 251
        sf = torch.arange(ops.mxfp4_sf_bytes(*x.shape)) * (1 + int(q.sum()) % 97) % 241
        return q.to(torch.uint8), sf.to(torch.uint8)

    def rows(q, sf, n, k):
        s = _unswizzle(sf, n, k // 32).double().repeat_interleave(16, 1)
        return q.double() * s

    def linear(w, x, **_):
        return x.double()[:, ::2] @ rows(w.qdata, w.scale, w.out_features, w.in_features).T

    def ffn(up, down, x, **_):
        f = up.out_features // 2
        order = ops.swiglu_rows(f)
        chunked = torch.empty(2 * f, up.in_features // 2, dtype=torch.float64)
        chunked[order] = rows(up.qdata, up.scale, 2 * f, up.in_features)
        return x.double()[:, ::2] @ chunked.T

    monkeypatch.setattr(ops, "mxfp4_quantize", quantize)
    monkeypatch.setattr(mxfp4, "mxfp4_linear", linear)
    monkeypatch.setattr(mxfp4, "gated_ffn", ffn)
    return linear


CHANGES = [rewrite, rebind, replace]


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_shared_qkv_follows_its_weights(on_cpu, change, which):
    qkv, _, _ = modules()
    x = torch.randn(3, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    for seed in (20, 21):
        for got, m in zip(mxfp4.shared_qkv(*qkv, x), qkv):
            assert torch.equal(got, m(x))
        change(qkv[which] if change is replace else qkv[which].weight_mxfp4, seed)
    for got, m in zip(mxfp4.shared_qkv(*qkv, x), qkv):
        assert torch.equal(got, m(x))


@pytest.mark.parametrize("change", CHANGES)
def test_linear_ffn_follows_its_weight(on_cpu, change):
    _, up, down = modules()
    x = torch.randn(3, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    for seed in (30, 31):
        assert torch.equal(mxfp4.linear_ffn(up, down, x), on_cpu(up.weight_mxfp4, x))
        change(up if change is replace else up.weight_mxfp4, seed)
    assert torch.equal(mxfp4.linear_ffn(up, down, x), on_cpu(up.weight_mxfp4, x))


def test_replaced_weights_of_other_widths(on_cpu):
    """The modules' weights count, not the widths that the modules had."""
    qkv, up, down = modules()
    x = torch.zeros(1, K, dtype=torch.bfloat16)
    mxfp4.shared_qkv(*qkv, x)
    qkv[0].weight_mxfp4 = lin(136, K, 43).weight_mxfp4        # not in whole scale tiles
    assert mxfp4.shared_qkv(*qkv, x) is None
    down.weight_mxfp4 = lin(K, 128, 44).weight_mxfp4
    assert mxfp4.linear_ffn(up, down, x) is None
    up.weight_mxfp4 = lin(256, K, 45).weight_mxfp4
    assert torch.equal(mxfp4.linear_ffn(up, down, x), on_cpu(up.weight_mxfp4, x))


def test_copies_are_kept_and_changed_in_place(on_cpu):
    qkv, up, down = modules()
    x = torch.zeros(1, K, dtype=torch.bfloat16)

    def at():
        mxfp4.shared_qkv(*qkv, x)
        mxfp4.linear_ffn(up, down, x)
        return [t.data_ptr() for m, slot in ((qkv[0], "_fused"), (up, "_gated"))
                for t in (getattr(m, slot)[1].qdata, getattr(m, slot)[1].scale)]

    first, kept = at(), qkv[0]._fused
    assert at() == first and qkv[0]._fused is kept            # nothing changed: nothing done
    for change in (rewrite, rebind):
        change(qkv[1].weight_mxfp4, 40)
        change(up.weight_mxfp4, 41)
        assert at() == first                                  # a captured call may read them
    qkv[1] = lin(256, K, 42)
    assert len(mxfp4.shared_qkv(*qkv, x)) == 3 and qkv[0]._fused[1].out_features == 640


def test_copied_modules_follow_their_own_weights(on_cpu):
    qkv, up, down = modules()
    x = torch.randn(2, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    mxfp4.shared_qkv(*qkv, x)
    mxfp4.linear_ffn(up, down, x)
    other, up2 = copy.deepcopy(qkv), copy.deepcopy(up)
    rewrite(other[1].weight_mxfp4, 50)
    rewrite(up2.weight_mxfp4, 51)
    for ms in (qkv, other):
        for got, m in zip(mxfp4.shared_qkv(*ms, x), ms):
            assert torch.equal(got, m(x))
    for u in (up, up2):
        assert torch.equal(mxfp4.linear_ffn(u, down, x), on_cpu(u.weight_mxfp4, x))


@pytest.mark.parametrize("build", [True, False])
@pytest.mark.parametrize("change", [True, False])
def test_inference_mode(on_cpu, build, change):
    """Weights made and changed inside inference mode and outside."""
    x = torch.randn(2, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    with torch.inference_mode(build):
        qkv, up, down = modules()
        if build:                           # stored codes that count no versions
            w = qkv[2].weight_mxfp4
            w.qdata, w.scale = w.qdata.clone(), w.scale.clone()
    for seed in (60, 61):
        for mode in (True, False):
            with torch.inference_mode(mode):
                for got, m in zip(mxfp4.shared_qkv(*qkv, x), qkv):
                    assert torch.equal(got, m(x))
                assert torch.equal(mxfp4.linear_ffn(up, down, x), on_cpu(up.weight_mxfp4, x))
        with torch.inference_mode(build or change):
            rewrite(qkv[2].weight_mxfp4, seed)
            rewrite(up.weight_mxfp4, seed + 5)


# ---------------------------------------------------------------- GPU
def same(qkv, ff, x, monkeypatch):
    monkeypatch.setenv("H3_NVFP4", "1")
    up, down = ff.net[0].proj, ff.net[2]
    for fused in (mxfp4.shared_qkv(*qkv, x), gm.qkv_projection(*qkv, x)):
        for got, m in zip(fused, qkv):
            assert torch.equal(got, m(x))
    w = up.weight_mxfp4
    plain = mxfp4.gated_ffn(mxfp4.gated_up_weight(w.dequantize(torch.float32)), down.weight_mxfp4, x)
    for got in (mxfp4.linear_ffn(up, down, x), gm.ffn(ff, x)):
        assert torch.equal(got, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 40, 200])
def test_shims_follow_changed_weights(cuda, monkeypatch, m):
    qkv, up, down = modules(cuda)
    ff = FeedForward(up, down)
    x = torch.randn(m, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)
    same(qkv, ff, x, monkeypatch)
    for i, mod in enumerate((*qkv, up)):
        w = mod.weight_mxfp4
        new = torch.randn(w.out_features, K, generator=torch.Generator().manual_seed(70 + i))
        ops.mxfp4_quantize(new.to(cuda), q_out=w.qdata, sf_out=w.scale)
        same(qkv, ff, x, monkeypatch)
        rebind(w, 80 + i, cuda)
        same(qkv, ff, x, monkeypatch)
        with torch.inference_mode():
            rewrite(w, 90 + i, cuda)
            same(qkv, ff, x, monkeypatch)


@pytest.mark.gpu
def test_captured_before_the_first_call(cuda):
    """A capture that comes first keeps nothing that only its replay fills, and
    its replays follow weights written in place."""
    qkv, up, down = modules(cuda)
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)
    for m in qkv:                                         # the operators themselves are loaded
        m(x)
    mxfp4.gated_ffn(mxfp4.MXFP4Weight(torch.zeros(2 * F, K, device=cuda)), down.weight_mxfp4, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (*mxfp4.shared_qkv(*qkv, x), mxfp4.linear_ffn(up, down, x))
    assert qkv[0]._fused is None and up._gated is None
    for seed in (100, 101):
        want = (*(m(x) for m in qkv), mxfp4.linear_ffn(up, down, x))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        for i, m in enumerate((*qkv, up)):
            rewrite(m.weight_mxfp4, seed + 10 * i, cuda)


@pytest.mark.gpu
def test_captured_with_kept_copies(cuda):
    """A captured call that reads the kept copies follows a change at the next
    call that is not captured."""
    qkv, up, down = modules(cuda)
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)

    def call():
        return (*mxfp4.shared_qkv(*qkv, x), mxfp4.linear_ffn(up, down, x))

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for change in (rewrite, rebind):
        for i, m in enumerate((*qkv, up)):
            change(m.weight_mxfp4, 110 + i, cuda)
        want = call()
        torch.empty(1 << 20, dtype=torch.uint8, device=cuda).fill_(255)   # what was freed
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_copies_are_there_for_other_streams(cuda):
    qkv, up, down = modules(cuda)
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)
    want = (*(m(x) for m in qkv),
            mxfp4.gated_ffn(mxfp4.gated_up_weight(up.weight_mxfp4.dequantize(torch.float32)),
                            down.weight_mxfp4, x))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        qkv[0]._fused = up._gated = None
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append((*mxfp4.shared_qkv(*qkv, x), mxfp4.linear_ffn(up, down, x)))
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.gpu
def test_compiled_callers_follow_their_weights(cuda):
    qkv, up, down = modules(cuda)
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)

    def call(x):
        q, k, v = mxfp4.shared_qkv(*qkv, x)
        return torch.cat([q, k, v], -1), mxfp4.linear_ffn(up, down, x)

    compiled = torch.compile(call, fullgraph=True, backend="aot_eager")
    for i in range(2):
        for got, want in zip(compiled(x), call(x)):
            assert torch.equal(got, want)
        for j, m in enumerate((*qkv, up)):
            rewrite(m.weight_mxfp4, 120 + 10 * i + j, cuda)
    for got, want in zip(compiled(x), call(x)):
        assert torch.equal(got, want)
