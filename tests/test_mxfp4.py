"""MXFP4 quantization, products and the gated feed-forward against 64-bit
arithmetic, and their refusals."""
import ctypes

import pytest
import torch

from h3_engine_b200 import _lib, mxfp4, ops
from tests import mx_ref as ref

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


# ---------------------------------------------------------------- CPU: refusals, schemas
def test_host_checks_refuse_without_a_gpu():
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    q = lib.h3b_mxfp4_quantize
    assert q(p, 0, 4, 48, 48, p, p, None) == 1            # K % 32
    assert q(p, 3, 4, 64, 64, p, p, None) == 1            # element type
    assert q(p, 0, 4, 64, 32, p, p, None) == 1            # row stride below K
    assert q(p, 0, -1, 64, 64, p, p, None) == 1
    assert q(None, 0, 4, 64, 64, p, p, None) == 1
    assert q(odd, 0, 4, 64, 64, p, p, None) == 2
    assert q(p, 0, 4, 64, 68, p, p, None) == 2            # rows not 16-byte aligned
    assert q(None, 0, 0, 64, 64, None, None, None) == 0   # no rows: nothing to do
    d = lib.h3b_mxfp4_dequantize
    assert d(p, p, 4, 40, p, 0, 40, None) == 1
    assert d(p, p, 4, 64, p, 0, 32, None) == 1
    assert d(p, p, 4, 64, odd, 0, 64, None) == 2
    g = lib.h3b_mxfp4_gemm
    assert g(p, p, 4, p, p, 12, 64, None, 0, None, 0, p, 0, 16, None) == 1    # N % 8
    assert g(p, p, 4, p, p, 16, 48, None, 0, None, 0, p, 0, 16, None) == 1    # K % 32
    assert g(p, p, 4, p, p, 16, 64, None, 2, None, 0, p, 0, 16, None) == 1    # activation
    assert g(p, p, 4, p, p, 16, 64, None, 0, None, 0, p, 2, 16, None) == 1    # fp32 result
    assert g(p, p, 4, p, p, 16, 64, None, 0, p, 8, p, 0, 16, None) == 1       # residual stride
    assert g(p, p, 4, p, p, 16, 64, odd, 0, None, 0, p, 0, 16, None) == 2
    assert g(p, p, 0, p, p, 16, 64, None, 0, None, 0, p, 0, 16, None) == 0
    lin = lib.h3b_mxfp4_linear
    assert lib.h3b_mxfp4_linear_ws(4, 16, 64) == 0        # few rows need none
    need = lib.h3b_mxfp4_linear_ws(20, 16, 64)
    assert need == 768 + 512                              # codes to 256 bytes, one scale tile
    assert lin(p, 0, 20, 64, p, p, 16, 64, None, 0, None, 0, p, 16, p, need - 1, None) == 1
    assert lin(p, 0, 20, 64, p, p, 16, 64, None, 0, None, 0, p, 16, odd, need, None) == 2
    assert lin(p, 0, 20, 32, p, p, 16, 64, None, 0, None, 0, p, 16, p, need, None) == 1   # ldx < K
    f = lib.h3b_mxfp4_ffn
    need = lib.h3b_mxfp4_ffn_ws(4, 64, 128)
    assert need == 2 * (256 + 512)
    assert f(p, 0, 4, 64, p, p, p, p, 64, 192, None, 0, p, 64, p, 1 << 30, None) == 1   # F % 128
    assert f(p, 0, 4, 64, p, p, p, p, 48, 128, None, 0, p, 48, p, 1 << 30, None) == 1   # N % 32
    assert f(p, 0, 4, 64, p, p, p, p, 64, 128, None, 0, p, 64, p, need - 1, None) == 1
    assert f(odd, 0, 4, 64, p, p, p, p, 64, 128, None, 0, p, 64, p, need, None) == 2


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=BF16)
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.ops.h3b.mxfp4_quantize(x)


@pytest.mark.parametrize("name,outs", [
    ("mxfp4_quantize", {"q", "sf"}), ("mxfp4_dequantize", {"out"}), ("mxfp4_gemm", {"out"}),
    ("mxfp4_linear", {"out"}), ("mxfp4_ffn", {"out"})])
def test_operators_declare_their_outputs(name, outs):
    schema = getattr(torch.ops.h3b, name + "_out").default._schema
    assert {a.name for a in schema.arguments
            if a.alias_info is not None and a.alias_info.is_write} == outs
    assert not schema.returns
    assert not any(a.alias_info for a in getattr(torch.ops.h3b, name).default._schema.arguments)


def test_operators_trace_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 96, dtype=BF16, device="cuda")
        q, sf = ops.mxfp4_quantize(x)
        assert q.shape == (15, 48) and sf.shape == (512,)
        assert ops.mxfp4_dequantize(q, sf, 15, 96, dtype=F32).shape == (15, 96)
        w = mxfp4.MXFP4Weight(torch.empty(64, 96, dtype=BF16, device="cuda"))
        assert mxfp4.mxfp4_linear(w, x).shape == (3, 5, 64)
        assert ops.mxfp4_gemm(q, sf, 15, w.qdata, w.scale, 64, 96, dtype=F16).dtype == F16
        up = mxfp4.gated_up_weight(torch.empty(256, 96, dtype=BF16, device="cuda"))
        down = mxfp4.MXFP4Weight(torch.empty(96, 128, dtype=BF16, device="cuda"))
        assert mxfp4.gated_ffn(up, down, x, out=torch.empty_like(x)).shape == x.shape


# ---------------------------------------------------------------- GPU
def mx_weight(n, k, cuda, seed=3):
    """A weight and the fp64 values that it stands for."""
    w = mxfp4.MXFP4Weight(rand(n, k, seed=seed, scale=k ** -0.5).to(BF16).to(cuda))
    s = ref.unblock(w.scale, n, k // 32)[:n, :k // 32]
    return w, ref.values(w.qdata, s)


def test_scales_must_be_aligned():
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 1)
    assert lib.h3b_mxfp4_quantize(p, 0, 4, 64, 64, p, odd, None) == 2
    assert lib.h3b_mxfp4_gemm(p, odd, 4, p, p, 16, 64, None, 0, None, 0, p, 0, 16, None) == 2
    assert lib.h3b_mxfp4_gemm(p, p, 4, p, odd, 16, 64, None, 0, None, 0, p, 0, 16, None) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (127, 96), (129, 160), (33, 1056),
                                    (5, 8224), (300, 2720)])
def test_quantize_is_exact(cuda, dtype, rows, k):
    x = rand(rows, k, seed=rows + k)
    x[:, ::7] *= 40
    x[rows // 2, :32] = 0
    x = x.to(dtype)
    q, sf = ops.mxfp4_quantize(x.to(cuda))
    want, s = ref.quantize(x)
    got = ref.unblock(sf, rows, k // 32)
    assert torch.equal(got[:rows, :k // 32], s)
    assert not got[rows:].any() and not got[:, k // 32:].any()       # padding is zero
    assert torch.equal(ref.values(q, s), want)
    for out in (BF16, F32):
        back = ops.mxfp4_dequantize(q, sf, rows, k, dtype=out)
        assert torch.equal(back.cpu().double(), want)


@pytest.mark.gpu
def test_quantize_ties_and_extremes(cuda):
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.999, 6.0, 7.9])
    x = torch.zeros(6, 64)
    x[0, :10], x[0, 31] = mids, 4.0          # unit 1: every tie, values up to 6 and beyond
    x[1, :10], x[1, 31] = -mids, -7.99
    x[2, :10] = mids * 2.0 ** -130           # subnormal block maximum in fp32
    x[3, 0], x[3, 1] = torch.finfo(F32).max, -1.0
    x[4, 0] = 2.0 ** -149
    x[5, 32:] = 2.0 ** 127
    q, sf = ops.mxfp4_quantize(x.to(cuda))
    want, s = ref.quantize(x)
    assert torch.equal(ref.unblock(sf, 6, 2)[:6, :2], s)
    assert torch.equal(ref.values(q, s), want)
    assert torch.equal(ops.mxfp4_dequantize(q, sf, 6, 64, dtype=F32).cpu().double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_non_finite_blocks_become_nan(cuda, dtype):
    x = rand(3, 96)
    x[0, 5], x[1, 40], x[2, 95] = float("inf"), float("nan"), float("-inf")
    q, sf = ops.mxfp4_quantize(x.to(dtype).to(cuda))
    back = ops.mxfp4_dequantize(q, sf, 3, 96, dtype=F32).cpu().view(3, 3, 32)
    bad = torch.eye(3, dtype=torch.bool)
    assert torch.isnan(back[bad]).all() and torch.isfinite(back[~bad]).all()


@pytest.mark.gpu
def test_quantize_strided_and_batched_inputs(cuda):
    wide = rand(2, 5, 200).to(BF16).to(cuda)
    for view in (wide[..., 8:136], wide[..., 3:131], wide.transpose(0, 1)[..., :64],
                 wide[0, :1, :96].expand(4, 96)):
        q, sf = ops.mxfp4_quantize(view)
        r = view.reshape(-1, view.shape[-1])
        want, s = ref.quantize(r)
        assert torch.equal(ref.values(q, ref.unblock(sf, *r.shape[:1], r.shape[1] // 32)
                                      [:r.shape[0], :r.shape[1] // 32]), want)
    # rows whose base or stride allows 16-byte accesses but not 32-byte ones
    for dtype in (BF16, F16, F32):
        base = rand(7, 24 + 320, seed=3).to(dtype).to(cuda)
        for view in (base[:, 8:8 + 320], base[:, 24:24 + 288]):
            q, sf = ops.mxfp4_quantize(view)
            k = view.shape[1]
            want, s = ref.quantize(view)
            assert torch.equal(ref.values(q, ref.unblock(sf, 7, k // 32)[:7, :k // 32]), want)
            out = torch.full((7, 24 + 320), 3.0, dtype=dtype, device=cuda)
            back = ops.mxfp4_dequantize(q, sf, 7, k, out=out[:, 8:8 + k])
            exact = want if dtype == F32 else want.to(dtype).double()
            assert torch.equal(back.cpu().double(), exact)
            assert (out[:, :8] == 3).all() and (out[:, 8 + k:] == 3).all()
    q, sf = ops.mxfp4_quantize(wide[:, :0, :64])
    assert q.shape == (0, 32) and sf.numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (2, 264, 96), (8, 128, 2720), (9, 136, 64), (16, 128, 256), (17, 520, 160),
                                   (33, 128, 2720), (64, 72, 512), (128, 1000, 1088),
                                   (129, 256, 64), (200, 392, 352), (513, 1032, 416),
                                   (257, 136, 4128), (384, 264, 4352)])
def test_linear_against_64_bits(cuda, dtype, m, n, k):
    x = rand(m, k, seed=m).to(dtype)
    w, wv = mx_weight(n, k, cuda)
    b, r = rand(n, seed=5).to(dtype), rand(m, n, seed=6).to(dtype)
    y, dy = ref.product(ref.quantize(x)[0], wv)
    h = ref.half_step(dtype)
    got = mxfp4.mxfp4_linear(w, x.to(cuda))
    assert got.dtype == dtype
    assert ((got.cpu().double() - y).abs() <= dy + h * (y.abs() + dy) + 1e-7).all()
    # bias, GELU (slope at most 1.13) and residual: their fp32 roundings, then the type's
    z = y + b.double()
    want = ref.gelu(z) + r.double()
    off = 1.13 * (dy + 2.0 ** -24 * z.abs()) + 2.0 ** -21 * (z.abs() + r.double().abs())
    got = mxfp4.mxfp4_linear(w, x.to(cuda), bias=b.to(cuda), act="gelu", residual=r.to(cuda))
    assert ((got.cpu().double() - want).abs() <= off + h * (want.abs() + off) + 1e-7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 140])
def test_activations_saturate(cuda, m):
    """GELU and the gate far out on both sides: v or 0, never NaN."""
    k, big = 64, 500.0
    x = torch.zeros(m, k, dtype=BF16)
    x[:, 0] = 1
    rows = torch.tensor([big, -big, 30.0, -30.0, 0.0, 6.0, -6.0, 1.0])   # products, exact
    w = torch.zeros(8, k)
    w[:, 0] = rows
    wv, _ = ref.quantize(w)
    got = mxfp4.mxfp4_linear(mxfp4.MXFP4Weight(w.to(BF16).to(cuda)), x.to(cuda), act="gelu")
    want = ref.gelu(wv[:, 0]).expand(m, 8)
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
    f, d = 128, 64
    up = torch.zeros(2 * f, k)
    up[:f, 0], up[f:, 0] = 1.0, rows.repeat(16)
    down = torch.eye(d, f)
    h, dh = ref.swiglu_bounded(torch.ones(1, f).double(), torch.zeros(1, f).double(),
                               ref.quantize(up[f:])[0][:, 0][None], torch.zeros(1, f).double())
    hq, far = ref.quantize_bounded(h, dh)
    got = mxfp4.gated_ffn(mxfp4.gated_up_weight(up.to(BF16).to(cuda)),
                          mxfp4.MXFP4Weight(down.to(BF16).to(cuda)), x.to(cuda)).cpu().double()
    assert ((got - hq[:, :d]).abs() <= far[:, :d] + 2.0 ** -8 * hq[:, :d].abs() + 1e-6).all()


@pytest.mark.gpu
def test_gemm_takes_quantized_operands(cuda):
    m, n, k = 150, 136, 224
    x = rand(m, k).to(BF16).to(cuda)
    w, _ = mx_weight(n, k, cuda)
    q, sf = ops.mxfp4_quantize(x)
    got = ops.mxfp4_gemm(q, sf, m, w.qdata, w.scale, n, k)
    assert torch.equal(got, mxfp4.mxfp4_linear(w, x))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 150])
def test_linear_views_outputs_and_nan_rows(cuda, m):
    n, k = 136, 288
    w, wv = mx_weight(n, k, cuda)
    big = rand(m, 3, k, seed=9).to(BF16).to(cuda)
    x = big[:, 1]
    out = torch.full((m + 2, 2 * n), 7.0, dtype=BF16, device=cuda)
    got = mxfp4.mxfp4_linear(w, x, out=out[1:m + 1, n:])
    assert got.data_ptr() == out[1:m + 1, n:].data_ptr()
    assert torch.equal(got, mxfp4.mxfp4_linear(w, x.contiguous()))
    assert (out[0] == 7).all() and (out[m + 1] == 7).all() and (out[:, :n] == 7).all()
    x3 = big[:, 1].unsqueeze(1)
    assert torch.equal(mxfp4.mxfp4_linear(w, x3), got.unsqueeze(1))
    assert mxfp4.mxfp4_linear(w, big[0, 0]).shape == (n,)
    assert mxfp4.mxfp4_linear(w, big[:0, 0]).shape == (0, n)
    y = x.clone()
    y[m - 1, 3] = float("nan")
    z = mxfp4.mxfp4_linear(w, y)
    assert torch.isnan(z[m - 1]).all() and torch.equal(z[:m - 1], got[:m - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,d,f", [(1, 32, 128), (3, 288, 384), (16, 256, 256), (40, 160, 512),
                                   (129, 544, 256), (260, 96, 640), (150, 4128, 128),
                                   (200, 64, 4224)])
def test_gated_ffn_against_64_bits(cuda, dtype, m, d, f):
    x, r = rand(m, d, seed=m).to(dtype), rand(m, d, seed=2).to(dtype)
    wu = rand(2 * f, d, seed=11, scale=d ** -0.5).to(BF16)
    up = mxfp4.gated_up_weight(wu.to(cuda))
    down, dv = mx_weight(d, f, cuda, seed=12)
    uv = ref.quantize(wu)[0]
    xq = ref.quantize(x)[0]
    v, ev = ref.product(xq, uv[:f])
    g, eg = ref.product(xq, uv[f:])
    h, dh = ref.swiglu_bounded(v, ev, g, eg)
    hq, far = ref.quantize_bounded(h, dh)
    y, dy = ref.product(hq, dv)
    dy = dy + far @ dv.abs().T
    for res in (None, r):
        want = y if res is None else y + res.double()
        off = dy + (0 if res is None else 2.0 ** -24 * want.abs())
        got = mxfp4.gated_ffn(up, down, x.to(cuda), residual=None if res is None else res.to(cuda))
        assert got.dtype == dtype
        assert ((got.cpu().double() - want).abs()
                <= off + ref.half_step(dtype) * (want.abs() + off) + 1e-7).all()
    # the bound is not vacuous: most hidden values are away from every boundary.
    # It covers d steps of 2^-23 of sum |x w|, about d^1.5 2^-23 of a typical
    # value: 3 % of it, a sixteenth of an E2M1 step on each side, at d = 4128.
    assert (far == 0).double().mean() > (0.9 if d < 1024 else 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [8, 9, 16, 17, 24, 25, 32, 33])
@pytest.mark.parametrize("n,k", [(136, 512), (520, 416), (264, 4128), (1024, 32)])
def test_rows_quantized_in_the_product_or_before(cuda, m, n, k):
    """The linear gives the bits of a quantization and a product, whichever kernel
    quantizes the rows (few rows of short K: the product's own)."""
    w = mxfp4.MXFP4Weight(rand(n, k, seed=13, scale=0.2).to(BF16).to(cuda))
    buf = rand(m, k + 16, seed=14).to(BF16).to(cuda)
    x, bias = buf[:, 8:8 + k], rand(n, seed=15).to(BF16).to(cuda)
    got = mxfp4.mxfp4_linear(w, x, bias=bias, act="gelu")
    q, sf = ops.mxfp4_quantize(x)
    want = ops.mxfp4_gemm(q, sf, m, w.qdata, w.scale, n, k, bias=bias, act=ops.ACT_GELU_TANH)
    assert torch.equal(got, want)
    if n % 128 == 0 and k % 32 == 0:
        up = mxfp4.gated_up_weight(rand(2 * n, k, seed=16, scale=0.2).to(BF16).to(cuda))
        down = mxfp4.MXFP4Weight(rand(k, n, seed=17, scale=0.2).to(BF16).to(cuda))
        one = mxfp4.gated_ffn(up, down, x)
        rows = torch.cat([mxfp4.gated_ffn(up, down, x[i:i + 1]) for i in range(m)])
        assert torch.equal(one, rows)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda):
    """The last rows of more than 2^31 values, there and back, and as a product."""
    m, k, last = 65600, 32832, 40
    x = torch.zeros(m, k, dtype=BF16, device=cuda)
    tail = rand(last, k, seed=11).to(BF16)
    x[m - last:] = tail.to(cuda)
    q, sf = ops.mxfp4_quantize(x)
    qt, st = ops.mxfp4_quantize(tail.to(cuda))
    assert torch.equal(q[m - last:], qt) and not q[:m - last].any()
    back = ops.mxfp4_dequantize(q, sf, m, k, out=x)
    assert torch.equal(back[m - last:], ops.mxfp4_dequantize(qt, st, last, k))
    w = mxfp4.MXFP4Weight(rand(8, k, seed=12).to(BF16).to(cuda))
    got = ops.mxfp4_gemm(q, sf, m, w.qdata, w.scale, 8, k)
    want = back[m - last:].double() @ w.dequantize(torch.float32).double().T
    # exact products summed in fp32: k 2^-23 of the sum of their magnitudes, then bf16
    size = back[m - last:].double().abs() @ w.dequantize(torch.float32).double().abs().T
    assert ((got[m - last:].double() - want).abs()
            <= k * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all()
    assert not got[:m - last].any()


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    w, _ = mx_weight(64, 64, cuda)
    x = torch.zeros(4, 64, dtype=BF16, device=cuda)
    with pytest.raises(TypeError):
        mxfp4.mxfp4_linear(w, x.float())
    with pytest.raises(TypeError):
        ops.mxfp4_quantize(x.double())
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x[:, :32])
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x[:, :40])
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, act="relu")
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, bias=torch.zeros(64, device=cuda))
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, residual=x[:3])
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, out=torch.empty(4, 32, dtype=BF16, device=cuda))
    with pytest.raises(ValueError):
        mxfp4.mxfp4_linear(w, x, out=torch.empty(64, 4, dtype=BF16, device=cuda).t())
    with pytest.raises(ValueError):
        ops.mxfp4_linear(x, w.qdata[:32], w.scale, 64, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_linear(x, w.qdata, w.scale[:-1], 64, 64)
    with pytest.raises(ValueError):
        mxfp4.MXFP4Weight(torch.zeros(12, 64, dtype=BF16, device=cuda))
    with pytest.raises(ValueError):
        mxfp4.gated_ffn(w, w, x)
