"""CPU: the entry points of 4-bit microscaled tensors, layers and the norms around a block refuse what they cannot take, without a GPU."""
import ctypes

import pytest
import torch

from shrew_b200 import Fp4Format, Fp4Linear, Fp4Tensor, Norm, NormKind, ShrewError, dequantize_fp4, quantize_fp4, residual_norm
from shrew_b200 import _lib


def test_null_handles_are_rejected():
    L, h = _lib.lib(), ctypes.c_void_p()
    assert L.shrewq_quantize_fp4(None, None, _lib.F32, 1, 32, 32, 0, None, 0, None, None) == _lib.ERR_INVALID_ARG
    assert L.shrewq_dequantize_fp4(None, None, None, None, 1, 32, 0, _lib.F32, None) == _lib.ERR_INVALID_ARG
    assert L.shrewq_linear_create_fp4(None, None, None, None, None, 1, 32, 0, 0, 1.0, ctypes.byref(h)) == _lib.ERR_INVALID_ARG
    assert not h.value
    assert L.shrewq_residual_norm(None, None) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("fmt", [Fp4Format.Mx, Fp4Format.Nv])
@pytest.mark.parametrize("call", ["quantize", "dequantize", "layer", "norm"])
def test_tensors_of_the_host_are_rejected(fmt, call):
    x = torch.zeros(4, 64)
    g = torch.ones(1) if fmt is Fp4Format.Nv else None
    t = Fp4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4 if g is not None else 2, dtype=torch.uint8), g, [4, 64], torch.float32, fmt)
    calls = {"quantize": lambda: quantize_fp4(x, fmt), "dequantize": lambda: dequantize_fp4(t), "layer": lambda: Fp4Linear(t),
             "norm": lambda: residual_norm(x, x, pre=Norm(NormKind.Rms, None))}
    with pytest.raises(ShrewError) as e:
        calls[call]()
    assert e.value.code == _lib.ERR_NO_DEVICE
