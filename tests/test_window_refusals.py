"""Refusals of the windowed-attention operators at the ends of their ranges."""
import ctypes

import pytest
import torch

from h3_engine_b200 import _lib, ops

BF16 = torch.bfloat16
LARGE = float(torch.finfo(torch.float32).max)


def test_a_scale_whose_exponents_overflow_is_refused():
    """The kernels work in log2 units: scale * log2(e) has to be a number too."""
    lib = _lib.lib()
    p = ctypes.c_void_p(1 << 20)
    one, zero = (ctypes.c_int32 * 1)(4), (ctypes.c_int32 * 1)(0)
    st = (ctypes.c_int64 * 3)(128, 128, 128)
    for scale in (LARGE, LARGE / 1.4):
        assert lib.h3b_attention_window(p, 4, 128, p, 128, p, 128, 4, 0, 1, 1, 128, zero, one, zero,
                                        one, 1, 0, 0, 0, 0, scale, p, 128, None, 0, None) == 1
        assert lib.h3b_attention_window_decode(p, st, p, st, p, st, p, 1, 4, 1, 0, 1, 1, 128, 0, 0,
                                               0, 1, scale, p, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [LARGE, LARGE / 1.4, 1e300, 1e-300, float("inf"), -1.0])
def test_scales_are_refused_as_fp32(cuda, scale):
    x = torch.zeros(8, 128, dtype=BF16, device=cuda)
    c = x.view(1, 8, 1, 128)
    n = torch.tensor([8], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        ops.attention_window(x, x, x, 1, 128, [0, 8], scale=scale)
    with pytest.raises(ValueError):
        ops.attention_window_decode(c[:, :1], c, c, n, scale=scale)


@pytest.mark.gpu
def test_the_largest_scale(cuda):
    """Equal logits at the largest scale that is taken: the mean of the values."""
    x = torch.zeros(8, 128, dtype=BF16, device=cuda)
    v = torch.arange(8, dtype=BF16, device=cuda)[:, None].expand(8, 128).contiguous()
    c, cv = x.view(1, 8, 1, 128), v.view(1, 8, 1, 128)
    n = torch.tensor([8], dtype=torch.int32, device=cuda)
    assert (ops.attention_window(x, x, v, 1, 128, [0, 8], scale=LARGE / 1.45) == 3.5).all()
    assert (ops.attention_window_decode(c[:, :1], c, cv, n, scale=LARGE / 1.45) == 3.5).all()


def decode(B, n_new, H, kv):
    p = ctypes.c_void_p(1 << 20)
    st = (ctypes.c_int64 * 3)(128, 128, 128)
    return _lib.lib().h3b_attention_window_decode(p, st, p, st, p, st, p, B, 4, n_new, 0, H, kv, 128,
                                                  0, 0, 0, 1, 0.1, p, None)


def test_decode_sizes_beyond_the_grid_are_refused_before_a_launch():
    for args in ((65536, 1, 1, 1), (1, 65536, 1, 1), (1, 16384, 128, 128), (1, 1, 65536, 65536)):
        assert decode(*args) == 1, args


@pytest.mark.gpu
def test_decode_sizes(cuda):
    """The largest batch and the largest number of rows, and one more of each."""
    def call(B, n, H, kv, d=64):
        q = torch.ones(1, 1, 1, 1, dtype=BF16, device=cuda).expand(B, n, H, d)
        k = torch.ones(B, 1, kv, d, dtype=BF16, device=cuda)
        length = torch.ones(B, dtype=torch.int32, device=cuda)
        return ops.attention_window_decode(q.contiguous(), k, k, length, causal=False)

    for args in ((65535, 1, 1, 1), (1, 65535, 16, 1), (1, 1, 65535, 65535)):
        assert (call(*args) == 1).all()
    for args in ((65536, 1, 1, 1), (1, 65536, 1, 1), (1, 65535, 17, 1), (1, 1, 65536, 65536)):
        with pytest.raises(ValueError):
            call(*args)


@pytest.mark.gpu
def test_head_dims_without_a_scale_of_their_own(cuda):
    x = torch.zeros(8, 128, dtype=BF16, device=cuda)
    for d in (0, -2, -64):
        with pytest.raises(ValueError):
            ops.attention_window(x, x, x, 1, d, [0, 8])
    c = torch.zeros(1, 8, 1, 0, dtype=BF16, device=cuda)
    with pytest.raises(ValueError):
        ops.attention_window_decode(c[:, :1], c, c, torch.ones(1, dtype=torch.int32, device=cuda))
