// Facts of a 4-bit weight tensor that its kernels need, in device memory that the handle owns.
#pragma once

namespace shrewq {

struct Fp4Params {
    float tensor_scale;      // NV; 1 for MX
    float x_scale;           // tensor scale of quantized activations (NV), else 1
    int max_byte, min_byte;  // MX: range of the scale bytes (NaN apart)
};

}  // namespace shrewq
