"""shrew_b200 — B200-native INT8 quantization path for Shrew (quantize / dequantize /
quantized Linear forward), hand-written sm_100a kernels behind a C ABI.

The names re-exported here are the ones the reference's facade crate re-exports for this
path (crates/shrew/src/lib.rs:120-124)."""
from .quantize import (  # noqa: F401
    Linear,
    QuantBits,
    QuantConfig,
    QuantGranularity,
    QuantMode,
    QuantStats,
    QuantizedLinear,
    QuantizedTensor,
    ShrewError,
    dequantize_tensor,
    quantization_stats,
    quantize_named_parameters,
    quantize_tensor,
    quantize_tensors,
)
from .block import GatedMlp, Norm, NormKind, residual_norm, run_blocks  # noqa: F401
from .fp4 import Fp4Format, Fp4Linear, Fp4Tensor, dequantize_fp4, quantize_fp4  # noqa: F401
