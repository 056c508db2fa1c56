"""4-bit microscaled floating point: quantization, dequantization and Linear layers over the codes.

Beyond the reference, whose 4-bit type is an integer with one scale a tensor or channel (crates/shrew/src/quantize.rs:51-61): E2M1
codes with a scale for every block along a row, the formats that a B200's block-scaled tensor cores multiply directly.

    Mx   blocks of 32, scales that are powers of two (E8M0)
    Nv   blocks of 16, E4M3 scales, one f32 scale for the tensor

Same manner as `quantize`: torch CUDA tensors in and out, work on torch's current stream, no CPU path.  The exact rules are in
include/shrewq.h.
"""
from __future__ import annotations

import ctypes
import enum
from dataclasses import dataclass
from typing import List, Optional

import torch

from . import _lib
from . import quantize as _q
from ._lib import ShrewError
from .quantize import Device, QuantizedLinear, _ptr, _rows_cols

__all__ = ["Fp4Format", "Fp4Tensor", "quantize_fp4", "dequantize_fp4", "Fp4Linear"]


class Fp4Format(enum.Enum):
    Mx = _lib.FP4_MX
    Nv = _lib.FP4_NV

    @property
    def block(self) -> int:
        """Values that share a scale."""
        return 32 if self is Fp4Format.Mx else 16


def _ext():
    return _q._host or _q._load_host()


@dataclass
class Fp4Tensor:
    """A quantized tensor.  rows = shape[0], cols = product(shape[1..]), padded to kp = a multiple of 32."""
    codes: torch.Tensor                    # uint8 [rows, kp / 2], the even column in the low nibble
    scales: torch.Tensor                   # uint8 [rows, kp / format.block]: E8M0 or E4M3 bytes
    tensor_scale: Optional[torch.Tensor]   # Nv: one float32 on the device; Mx: None
    shape: List[int]
    original_dtype: torch.dtype
    format: Fp4Format

    def numel(self) -> int:
        n = 1
        for s in self.shape:
            n *= int(s)
        return n

    def size_bytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (4 if self.tensor_scale is not None else 0)

    def compression_ratio(self) -> float:
        """Against f32, as QuantizedTensor.compression_ratio; 1.0 for an empty tensor."""
        return (self.numel() * 4) / self.size_bytes() if self.numel() else 1.0


def quantize_fp4(tensor: torch.Tensor, format: Fp4Format = Fp4Format.Mx, tensor_scale: Optional[torch.Tensor] = None) -> Fp4Tensor:
    """An f32, bf16 or f16 CUDA tensor as 4-bit codes with block scales along its rows (shrewq_quantize_fp4).  `tensor_scale` (Nv
    only): one float32 on the device, 2^-126 or more; by default the smallest power of two that brings the largest block scale under E4M3's
    largest value, found in a pass of its own."""
    if not tensor.is_cuda:
        Device.get(tensor.device)    # raises: CUDA devices only
    return Fp4Tensor(*_ext().quantize_fp4(tensor, format.value, tensor_scale), tensor.dtype, format)


def dequantize_fp4(t: Fp4Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """code * scale (* tensor scale) as a tensor of t's shape, of its original dtype or `out_dtype` (f32, bf16, f16)."""
    if not t.codes.is_cuda:
        Device.get(t.codes.device)
    return _ext().dequantize_fp4(t.codes, t.scales, t.tensor_scale, t.shape, t.format.value, out_dtype or t.original_dtype)


class Fp4Linear(QuantizedLinear):
    """A Linear over 4-bit microscaled weights, with the surface of QuantizedLinear: forward, forward_gate_up_silu, forward_host and
    the Module methods.  Any in_features; activations f32 or bf16.

    quantize_activations=False: x . dequant(W)^T + bias, products exact, sums in f32.
    quantize_activations=True: the rows of x are first quantized to the weights' format (Nv with `activation_scale` as their
    tensor scale, which nothing else uses) and multiplied code by code on the block-scaled tensor cores.

    Most calls with more than a few tokens, and all that quantize activations, use a workspace of the device's context
    (include/shrewq.h, shrewq_linear_create_fp4): calls on different streams, and replays of captured ones, have to be ordered."""

    def __init__(self, weight: Fp4Tensor, bias: Optional[torch.Tensor] = None, quantize_activations: bool = False,
                 activation_scale: float = 1.0):
        if len(weight.shape) != 2:
            raise ShrewError(_lib.ERR_INVALID_ARG, "Fp4Linear needs a rank-2 weight [out,in]")
        rows, cols = _rows_cols(weight.shape)
        kp = (cols + 31) // 32 * 32
        dev = weight.codes.device
        for t, need, what in ((weight.codes, rows * kp // 2, "codes"), (weight.scales, rows * kp // weight.format.block, "scales")):
            if t.dtype is not torch.uint8 or t.numel() != need or not t.is_contiguous() or t.device != dev:
                raise ShrewError(_lib.ERR_INVALID_ARG, f"Fp4Linear: {what} must be {need} contiguous uint8 values on one device")
        g = weight.tensor_scale
        if (g is not None) != (weight.format is Fp4Format.Nv) or (g is not None and (g.dtype is not torch.float32 or g.numel() != 1 or g.device != dev)):
            raise ShrewError(_lib.ERR_INVALID_ARG, "Fp4Linear: an Nv weight has one float32 tensor scale on its device, an Mx weight none")
        self.weight_q, self.bias = weight, bias
        self.out_features, self.in_features = rows, cols
        self.quantize_activations = bool(quantize_activations)
        self.device = Device.get(dev)
        self._bias_flat = None
        if bias is not None:
            if bias.numel() != rows:
                raise ShrewError(_lib.ERR_INVALID_ARG, "bias must have out_features elements")
            self._bias_flat = bias.detach().reshape(-1).to(device=dev, dtype=torch.float32).contiguous()
        h = ctypes.c_void_p()
        self.device.bind_stream()
        rc = _lib.lib().shrewq_linear_create_fp4(self.device.handle, _ptr(weight.codes), _ptr(weight.scales), _ptr(g), _ptr(self._bias_flat),
                                                 rows, cols, weight.format.value, int(self.quantize_activations), float(activation_scale),
                                                 ctypes.byref(h))
        _lib.check(rc, self.device.handle)
        self._h = h
        self._bind_host()

    def _bind_host(self) -> None:
        self._layer = _ext().Layer(self.device.handle.value, self._h.value, self.device.index, self.in_features, self.out_features)
        self._forward, self._gate_up = self._layer.forward, self._layer.gate_up_silu

    @classmethod
    def new(cls, weight: Fp4Tensor, bias: Optional[torch.Tensor] = None, **options) -> "Fp4Linear":
        return cls(weight, bias, **options)

    @classmethod
    def new_int4_packed(cls, *args, **kwargs):
        raise ShrewError(_lib.ERR_UNSUPPORTED, "Fp4Linear holds floating point codes; packed INT4 goes with QuantizedLinear")

    @classmethod
    def from_linear(cls, linear, format: Fp4Format = Fp4Format.Mx, **options) -> "Fp4Linear":
        """As QuantizedLinear.from_linear: params[0] is the weight, params[1] the bias if present."""
        params = list(linear.parameters())
        return cls(quantize_fp4(params[0].detach(), format), params[1].detach() if len(params) > 1 else None, **options)

    def __repr__(self) -> str:
        return (f"Fp4Linear(in_features={self.in_features}, out_features={self.out_features}, format={self.weight_q.format.name}, "
                f"quantize_activations={self.quantize_activations}, compression={self.weight_q.compression_ratio():.1f}x)")
