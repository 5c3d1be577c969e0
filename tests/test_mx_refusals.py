"""Outputs of the MXFP4 operators that are no rows at one stride."""
import pytest
import torch

from h3_engine_b200 import mxfp4

BF16 = torch.bfloat16


@pytest.mark.gpu
def test_outputs_that_are_no_rows_at_one_stride(cuda):
    g = torch.Generator().manual_seed(1)
    w = mxfp4.MXFP4Weight(torch.randn(64, 64, generator=g).to(BF16).to(cuda))
    up = mxfp4.gated_up_weight(torch.randn(256, 64, generator=g).to(BF16).to(cuda))
    down = mxfp4.MXFP4Weight(torch.randn(64, 128, generator=g).to(BF16).to(cuda))
    x = torch.randn(2, 3, 64, generator=g).to(BF16).to(cuda)
    for call in (lambda **kw: mxfp4.mxfp4_linear(w, x, **kw),
                 lambda **kw: mxfp4.gated_ffn(up, down, x, **kw)):
        want = call()
        for out in (torch.empty(3, 2, 64, dtype=BF16, device=cuda).transpose(0, 1),
                    torch.empty(2, 4, 64, dtype=BF16, device=cuda)[:, :3]):
            with pytest.raises(ValueError):
                call(out=out)
        out = torch.empty(2, 3, 128, dtype=BF16, device=cuda)[..., 64:]     # rows at 128
        assert call(out=out) is out and torch.equal(out, want)
        empty = torch.empty(0, 3, 64, dtype=BF16, device=cuda)
        assert mxfp4.mxfp4_linear(w, empty, out=torch.empty_like(empty)).shape == empty.shape
