"""MXFP4 products over more weight rows than a grid's second dimension has tiles."""
import pytest
import torch

from h3_engine_b200 import _lib, mxfp4, ops

BF16 = torch.bfloat16
LIMIT = 65535 * 128


def test_workspace_follows_the_kernel():
    ws = _lib.lib().h3b_mxfp4_linear_ws
    assert ws(1, LIMIT, 32) == ws(8, LIMIT, 32) == 0
    for m in (1, 8, 9):
        assert ws(m, LIMIT + 8, 32) == (m * 32 + 255) // 256 * 256 + 512
    assert ws(0, LIMIT + 8, 32) == ws(-1, LIMIT + 8, 32) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 20, 128, 129])
def test_linear_over_many_weight_rows(cuda, m):
    """The same values as over the weight's first and last rows alone, and 64 bits'."""
    sums = 40 * 2.0 ** -23 * 1e3       # 32 additions and GELU's steps, sums |x w| up to 1e3
    n, k, part = LIMIT + 128, 32, 4096
    g = torch.Generator(device=cuda).manual_seed(3)
    w = mxfp4.MXFP4Weight(torch.randn(n, k, generator=g, device=cuda, dtype=BF16))
    x = torch.randn(m, k, generator=g, device=cuda, dtype=BF16)
    bias = torch.randn(n, generator=g, device=cuda, dtype=BF16)
    out = mxfp4.mxfp4_linear(w, x, bias=bias, act="gelu")
    q, sf = ops.mxfp4_quantize(x)
    assert torch.equal(ops.mxfp4_gemm(q, sf, m, w.qdata, w.scale, n, k, bias=bias,
                                      act=ops.ACT_GELU_TANH), out)
    for a in (0, n - part):
        some = mxfp4.MXFP4Weight.from_packed(w.qdata[a:a + part], w.scale[a * 4:(a + part) * 4],
                                             part, k)
        want = mxfp4.mxfp4_linear(some, x, bias=bias[a:a + part], act="gelu")
        assert ((out[:, a:a + part].double() - want.double()).abs()      # half a step each
                <= 2 * 2.0 ** -8 * want.double().abs() + sums).all()
    for a in range(0, n, 1 << 20):                       # every column: fp32 of the values
        b = min(n, a + (1 << 20))
        some = mxfp4.MXFP4Weight.from_packed(w.qdata[a:b], w.scale[a * 4:b * 4], b - a, k)
        y = (ops.mxfp4_dequantize(q, sf, m, k, dtype=torch.float32)[-1:].double()
             @ some.dequantize(torch.float32).double().T + bias[a:b].double())
        y = torch.nn.functional.gelu(y, approximate="tanh")
        assert ((out[-1:, a:b].double() - y).abs() <= 2.0 ** -8 * y.abs() + sums).all()


@pytest.mark.gpu
def test_feed_forward_over_many_weight_rows(cuda):
    """One row of 129 rows' result: the down projection picks single values."""
    d, f = 32, LIMIT // 2 // 128 * 128 + 128
    g = torch.Generator(device=cuda).manual_seed(4)
    up = mxfp4.gated_up_weight(torch.randn(2 * f, d, generator=g, device=cuda, dtype=BF16))
    down = torch.zeros(d, f, dtype=BF16, device=cuda)
    down[torch.arange(d), torch.linspace(0, f - 1, d).long()] = 1
    down = mxfp4.MXFP4Weight(down)
    x = torch.randn(129, d, generator=g, device=cuda, dtype=BF16)
    want = mxfp4.gated_ffn(up, down, x)
    assert want.any() and torch.isfinite(want).all()
    for m in (1, 20):
        assert torch.equal(mxfp4.gated_ffn(up, down, x[:m]), want[:m])
