"""MXFP4 linears beside the NVFP4 ones of ``nvfp4.py``: E2M1 codes with one
power-of-two (E8M0) scale per 32 values of K and no tensor-wide scale.

Without a tensor-wide scale an activation is quantized in one pass, and the
gated feed-forward's up projection writes its hidden activation as MXFP4 from
its own epilogue.  Activations and results are bf16 or fp16, products
accumulate in fp32.  As for NVFP4 there is no CPU path: without a CUDA device
and the built library every entry point raises.
"""
from __future__ import annotations

import torch
from torch import nn

from . import ops, torch_ops
from .nvfp4 import _block_linears, _set_child, _swizzle, _unswizzle

MXFP4_BLOCK = ops.MX_BLOCK
DTYPES = (torch.bfloat16, torch.float16)      # of activations and results

_LINEAR = torch_ops.ext_op("mxfp4_linear")
_ACTS = {None: ops.ACT_NONE, "gelu": ops.ACT_GELU_TANH}


class MXFP4Weight:
    """A quantized ``nn.Linear`` weight ``[out_features, in_features]``:
    ``qdata`` u8 ``[N, K/2]`` (low nibble = even K) and ``scale`` the flat
    blocked E8M0 bytes the GEMM reads."""

    __slots__ = ("qdata", "scale", "out_features", "in_features")

    def __init__(self, weight: torch.Tensor):
        self.out_features, self.in_features = weight.shape
        if self.out_features % 8:
            raise ValueError(f"out_features = {self.out_features} must be a multiple of 8")
        # normal tensors in every mode: those of inference mode count no versions (_laid_out)
        with torch.inference_mode(False):
            self.qdata, self.scale = ops.mxfp4_quantize(weight.detach())

    @classmethod
    def from_packed(cls, qdata: torch.Tensor, scale: torch.Tensor, out_features: int,
                    in_features: int) -> "MXFP4Weight":
        """From stored codes and blocked scales (checked when they are used)."""
        w = cls.__new__(cls)
        w.qdata, w.scale = qdata, scale
        w.out_features, w.in_features = out_features, in_features
        return w

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return ops.mxfp4_dequantize(self.qdata, self.scale, self.out_features, self.in_features,
                                    dtype=dtype)

    def nbytes(self) -> int:
        return self.qdata.numel() + self.scale.numel()


def mxfp4_linear(w: MXFP4Weight, x: torch.Tensor, *, bias: torch.Tensor | None = None,
                 act: str | None = None, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(Q(x) @ w.T + bias) + residual`` in x's type (bf16 or fp16);
    ``act`` is None or "gelu" (tanh form)."""
    if act not in _ACTS:
        raise ValueError(f"unknown activation {act!r}")
    if out is None and x.is_cuda:         # single tokens: no call in between
        return _LINEAR(x, w.qdata, w.scale, w.out_features, w.in_features, bias, _ACTS[act],
                       residual)
    return ops.mxfp4_linear(x, w.qdata, w.scale, w.out_features, w.in_features, bias=bias,
                            act=_ACTS[act], residual=residual, out=out)


def gated_up_weight(weight: torch.Tensor) -> MXFP4Weight:
    """The fused [value | gate] up projection ``[2F, K]`` (the reference's chunk
    order) as the weight ``gated_ffn`` takes: rows in ``ops.swiglu_rows``
    order."""
    return MXFP4Weight(weight[ops.swiglu_rows(weight.shape[0] // 2).to(weight.device)])


def gated_ffn(up: MXFP4Weight, down: MXFP4Weight, x: torch.Tensor, *,
              residual: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(v * silu(g)) @ down.T + residual`` with ``[v | g] = Q(x) @ up.T``
    (``up`` from ``gated_up_weight``), in x's type."""
    f = up.out_features // 2
    if down.in_features != f or down.out_features != up.in_features or up.out_features % 2:
        raise ValueError(f"up [{up.out_features}, {up.in_features}] and down "
                         f"[{down.out_features}, {down.in_features}] do not form a feed-forward")
    return ops.mxfp4_ffn(x, up.qdata, up.scale, down.qdata, down.scale, up.in_features, f,
                         residual=residual, out=out)


class MXFP4Linear(nn.Module):
    """An MXFP4 linear, with or without bias."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        self.weight_mxfp4 = MXFP4Weight(linear.weight.data)
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.bias = None if linear.bias is None else nn.Parameter(linear.bias.data,
                                                                  requires_grad=False)
        self._fused = self._gated = None      # laid out once: shared_qkv, linear_ffn

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mxfp4_linear(self.weight_mxfp4, x, bias=self.bias)


def _laid_out(module: nn.Module, slot: str, ws: tuple, lay_out) -> MXFP4Weight:
    """``lay_out()``, a weight made of the weights ``ws``, kept in ``module.slot``
    until one of them has another tensor or, as the tensor's version tells, other
    contents.  (Writes that no version counts, through ``.data`` or by a graph's
    replay, are not seen.)

    A change is written into the kept tensors, which live as long as the module:
    a captured call goes on reading them, and follows at the next call that is not
    captured.  The device is waited for around that, and after the first layout,
    because calls on every stream read them.  Not kept is what would only be there
    after a replay or inside a compiled call, and what is made of tensors without
    versions (those of inference mode)."""
    if torch.compiler.is_compiling():
        return lay_out()
    kept = getattr(module, slot)
    if kept is not None and len(kept[0]) == len(ws):
        for w, (q, q_version, sf, sf_version, n, k) in zip(ws, kept[0]):
            if (w.qdata is not q or q._version != q_version or w.scale is not sf
                    or sf._version != sf_version or w.out_features != n or w.in_features != k):
                break
        else:
            return kept[1]
    sources = [t for w in ws for t in (w.qdata, w.scale)]
    if any(t.is_inference() for t in sources):
        return lay_out()
    made_of = [(w.qdata, w.qdata._version, w.scale, w.scale._version, w.out_features,
                w.in_features) for w in ws]
    on_gpu = sources[0].is_cuda
    with torch.inference_mode(False):
        w = lay_out()
        if on_gpu and torch.cuda.is_current_stream_capturing():
            return w
        if kept is not None:
            if on_gpu:
                torch.cuda.synchronize(sources[0].device)
            if all(a.shape == b.shape and a.device == b.device for a, b in
                   ((kept[1].qdata, w.qdata), (kept[1].scale, w.scale))):
                w.qdata, w.scale = kept[1].qdata.copy_(w.qdata), kept[1].scale.copy_(w.scale)
    if on_gpu:
        torch.cuda.current_stream(sources[0].device).synchronize()
    setattr(module, slot, (made_of, w))
    return w


def shared_qkv(to_q, to_k, to_v, x: torch.Tensor):
    """q, k and v projections from one quantization of ``x`` as one product over
    the weights concatenated along N (a second copy of them, kept on ``to_q`` and
    following them): None unless all three are ``MXFP4Linear`` of one input width,
    without bias, with output widths in whole 128-row scale tiles, and ``x`` is of
    a type they take."""
    mods = (to_q, to_k, to_v)
    if x.dtype not in DTYPES or not all(isinstance(m, MXFP4Linear) and m.bias is None
                                        for m in mods):
        return None
    ws = tuple(m.weight_mxfp4 for m in mods)
    k = ws[0].in_features
    if any(w.out_features % 128 or w.in_features != k for w in ws):
        return None
    fused = _laid_out(to_q, "_fused", ws, lambda: MXFP4Weight.from_packed(
        torch.cat([w.qdata for w in ws]), torch.cat([w.scale for w in ws]),
        sum(w.out_features for w in ws), k))
    return mxfp4_linear(fused, x).split([w.out_features for w in ws], -1)


def linear_ffn(up: "MXFP4Linear", down: "MXFP4Linear", x: torch.Tensor):
    """``gated_ffn`` of a feed-forward's two linears, ``up`` the fused
    [value | gate] projection in the reference's chunk order (a copy with its rows
    reordered is kept on ``up`` and follows it): None if ``gated_ffn`` does not
    take them."""
    w, wd = up.weight_mxfp4, down.weight_mxfp4
    f = wd.in_features
    if (up.bias is not None or down.bias is not None or f % 128 or w.out_features != 2 * f
            or wd.out_features != w.in_features or x.dtype not in DTYPES):
        return None

    def in_groups(t):        # rows in swiglu_rows order: groups of 64 values and 64 gates
        return t.view(2, f // 64, 64, -1).transpose(0, 1).reshape(2 * f, -1)

    def reordered():
        sf = _unswizzle(w.scale, 2 * f, w.in_features // MXFP4_BLOCK)
        return MXFP4Weight.from_packed(in_groups(w.qdata),
                                       _swizzle(in_groups(sf)).view(torch.uint8),
                                       2 * f, w.in_features)

    return gated_ffn(_laid_out(up, "_gated", (w,), reordered), wd, x)


@torch.no_grad()
def quantize_blocks(model) -> dict:
    """Swap the six block linears of every transformer block for MXFP4 ones, as
    ``nvfp4.quantize_blocks`` does for NVFP4."""
    slots = [(parent, name) for block in model.transformer_blocks
             for parent, name, _ in _block_linears(block)]
    for parent, name in slots:
        _set_child(parent, name, MXFP4Linear(parent._modules[name]))
    return {"linears_quantized": len(slots)}
