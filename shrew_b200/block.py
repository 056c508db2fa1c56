"""Around a quantized block: the norms before and after it, its gate and the residual scale in one kernel, and the gated MLP block
that runs between them.

The reference composes these from shrew-nn's norms and tensor operations; here they are one pass over the rows
(shrewq_residual_norm), and `GatedMlp` is the block of `QuantizedLinear.forward_gate_up_silu` and `forward` that a decoder runs.
"""
from __future__ import annotations

import enum
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from . import quantize as _q
from ._lib import ShrewError
from .quantize import Device, QuantizedLinear

__all__ = ["NormKind", "Norm", "residual_norm", "GatedMlp", "run_blocks"]


class NormKind(enum.Enum):
    Rms = _lib.NORM_RMS
    Layer = _lib.NORM_LAYER


class Norm:
    """The parameters of a norm over the last dimension; weight and bias (kept as contiguous f32) may be left out.

    Rms:   v / sqrt(mean(v^2) + eps) * weight + bias
    Layer: (v - mean) / sqrt(mean((v - mean)^2) + eps) * weight + bias"""

    def __init__(self, kind: NormKind = NormKind.Rms, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                 eps: float = 1e-5):
        if not eps >= 0.0:
            raise ShrewError(_lib.ERR_INVALID_ARG, "Norm: eps must not be negative")
        self.kind, self.eps = kind, float(eps)
        self.weight, self.bias = (None if t is None else t.detach().reshape(-1).to(torch.float32).contiguous() for t in (weight, bias))
        self._args = (kind.value, self.weight, self.bias, self.eps)


_NO_NORM = (_lib.NORM_NONE, None, None, 0.0)


def residual_norm(x: torch.Tensor, branch: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, *,
                  pre: Optional[Norm] = None, post: Optional[Norm] = None, residual_scale: float = 1.0, branch_scale: float = 1.0,
                  out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(r, h) with r = residual_scale * x + branch_scale * gate * post(branch) and h = pre(r), in one pass.

    x: the residual stream, [..., D], f32 or bf16; branch: the output of the block before, of its shape; gate, of branch's dtype: [D], or
    [..., 1], or of x's shape.  What is left out does nothing; h is None without `pre`.  r has x's dtype, h `out_dtype` (x's by
    default); both are rounded once from f32, h from the r before its rounding.  Without a branch and with residual_scale 1, r is x
    itself."""
    if not x.is_cuda:
        Device.get(x.device)    # raises: CUDA devices only
    return (_q._host or _q._load_host()).residual_norm(x, branch, gate, *(pre._args if pre else _NO_NORM), *(post._args if post else _NO_NORM),
                                                       residual_scale, branch_scale, out_dtype)


class GatedMlp:
    """A gated MLP block, down(silu(gate(h)) * up(h)), over quantized layers of any kind (QuantizedLinear, Fp4Linear), with the norm
    before it and, optionally, a norm after it, a gate and the residual scale:

        x -> residual_scale * x + branch_scale * channel_gate * post(down(silu(gate(pre(x))) * up(pre(x))))"""

    def __init__(self, gate: QuantizedLinear, up: QuantizedLinear, down: QuantizedLinear, pre: Norm, post: Optional[Norm] = None,
                 channel_gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, branch_scale: float = 1.0):
        if gate.in_features != up.in_features or gate.out_features != up.out_features or down.in_features != gate.out_features or \
                down.out_features != gate.in_features:
            raise ShrewError(_lib.ERR_INVALID_ARG, "GatedMlp: gate and up [ff, d] and down [d, ff] of one width d")
        self.gate, self.up, self.down = gate, up, down
        self.pre, self.post, self.channel_gate = pre, post, channel_gate
        self.residual_scale, self.branch_scale = residual_scale, branch_scale

    def block(self, h: torch.Tensor) -> torch.Tensor:
        """The branch alone: h [M, d], normalised, to [M, d]."""
        return self.down.forward(self.gate.forward_gate_up_silu(self.up, h))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [M, d] through the whole block: the new residual stream, of x's dtype."""
        return run_blocks([self], x)[0]

    __call__ = forward


def run_blocks(blocks: Sequence[GatedMlp], x: torch.Tensor, final: Optional[Norm] = None,
               act_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """x [M, d] through blocks one after the other: (residual stream, final(residual stream) or None).  Each block's end and the norm
    before the next (or `final`) are one kernel.  `act_dtype`: what the blocks compute in (x's dtype by default), so that an f32
    stream can feed bf16 products."""
    norms: List[Optional[Norm]] = [b.pre for b in blocks[1:]] + [final]
    if not blocks:
        return residual_norm(x, pre=final, out_dtype=act_dtype)
    _, h = residual_norm(x, pre=blocks[0].pre, out_dtype=act_dtype)
    for b, after in zip(blocks, norms):
        branch = b.block(h)
        gate = b.channel_gate
        if gate is not None and gate.dtype is not branch.dtype:
            gate = gate.to(branch.dtype)
        x, h = residual_norm(x, branch, gate, pre=after, post=b.post, residual_scale=b.residual_scale, branch_scale=b.branch_scale,
                             out_dtype=act_dtype or x.dtype)
    return x, h
