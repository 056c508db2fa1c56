// Launchers of the 4-bit floating point quantizer and dequantizer (device code and its description: fp4_kernels.cuh).
#include <cuda_fp16.h>

#include "fp4_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

size_t blocks_of(size_t threads_wanted, size_t cap) {
    const size_t b = (threads_wanted + kFp4Threads - 1) / kFp4Threads;
    return b < 1 ? 1 : (b > cap ? cap : b);
}

__global__ void fill_f32_kernel(float *p, float v) {
    pdl_launch_dependents();
    pdl_wait();
    *p = v;
}

int fill_f32(shrewq_ctx *ctx, float *p, float v) {
    SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(fill_f32_kernel, dim3(1), dim3(1), 0, ctx->stream, ctx->tuning.pdl != 0, p, v));
    ctx->launches += 1;
    return SHREWQ_OK;
}

template <typename T, bool NV>
int quantize_as(shrewq_ctx *ctx, const T *x, size_t rows, size_t cols, size_t ld, float *g, int find_g, uint32_t *codes, uint8_t *scales) {
    const bool pdl = ctx->tuning.pdl != 0;
    const bool aligned = (reinterpret_cast<uintptr_t>(x) % (8 * sizeof(T))) == 0;
    const bool flat = aligned && cols % 32 == 0 && (ld == cols || rows == 1);
    int source = kScaleGiven;
    if (NV && find_g) {
        const size_t grid = blocks_of((flat ? rows * cols / 8 : rows * ((cols + 7) / 8)) / 4, (size_t)ctx->sm_count * 8);
        source = (size_t)find_g > grid ? (int)grid : kScaleFound;
        if (source == kScaleFound && grid > 1) {
            const int rc = fill_f32(ctx, g, 0.0f);
            if (rc != SHREWQ_OK) return rc;
        }
        auto kern = flat ? fp4_tensor_scale_kernel<T, true> : fp4_tensor_scale_kernel<T, false>;
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(kern, dim3((unsigned)grid), dim3(kFp4Threads), 0, ctx->stream, pdl, x, rows, cols, ld, g, (int)(source > 0)));
        ctx->launches += 1;
    }
    constexpr int U = 4;
    const size_t groups = rows * cols / 8, want = (groups + kFp4Threads * U - 1) / (kFp4Threads * U);
    if (flat && want <= 0x7FFFFFFF) {
        const size_t grid = source != kScaleGiven && want > (size_t)ctx->sm_count * 6 ? (size_t)ctx->sm_count * 6 : want;
        auto kern = NV && source != kScaleGiven ? fp4_quantize_flat_kernel<T, NV, !NV, U> : fp4_quantize_flat_kernel<T, NV, true, U>;
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(kern, dim3((unsigned)grid), dim3(kFp4Threads), 0, ctx->stream, pdl, x, groups, g, source, codes, scales));
    } else {
        const size_t blocks = (cols + 31) / 32 * (NV ? 2 : 1), threads = (blocks * (NV ? 2 : 4) + 31) / 32 * 32;
        const int vec_ok = aligned && (ld * sizeof(T)) % (8 * sizeof(T)) == 0;
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(fp4_quantize_rows_kernel<T, NV>, dim3((unsigned)(rows < 0x7FFFFFFF ? rows : 0x7FFFFFFF)),
                                              dim3((unsigned)(threads < kFp4Threads ? threads : kFp4Threads)), 0, ctx->stream, pdl, x, rows, cols, ld,
                                              vec_ok, g, source, blocks, codes, scales));
    }
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <typename T>
int quantize_format(shrewq_ctx *ctx, const void *x, size_t rows, size_t cols, size_t ld, bool nv, float *g, int find_g, void *codes, void *scales) {
    uint32_t *c = static_cast<uint32_t *>(codes);
    uint8_t *s = static_cast<uint8_t *>(scales);
    return nv ? quantize_as<T, true>(ctx, static_cast<const T *>(x), rows, cols, ld, g, find_g, c, s)
              : quantize_as<T, false>(ctx, static_cast<const T *>(x), rows, cols, ld, nullptr, 0, c, s);
}

template <typename T, bool NV>
int dequantize_as(shrewq_ctx *ctx, const uint32_t *codes, const uint8_t *scales, const float *g, size_t rows, size_t cols, T *out) {
    const bool pdl = ctx->tuning.pdl != 0, aligned = (reinterpret_cast<uintptr_t>(out) % (8 * sizeof(T))) == 0;
    constexpr int U = 4;
    const size_t groups = rows * cols / 8, want = (groups + kFp4Threads * U - 1) / (kFp4Threads * U);
    if (aligned && cols % 32 == 0 && want <= 0x7FFFFFFF) {
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(fp4_dequantize_flat_kernel<T, NV, U>, dim3((unsigned)want), dim3(kFp4Threads), 0, ctx->stream, pdl, codes, scales,
                                              g, groups, out));
    } else {
        const size_t total = rows * ((cols + 7) / 8);
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(fp4_dequantize_rows_kernel<T, NV>, dim3((unsigned)blocks_of(total, (size_t)ctx->sm_count * 32)), dim3(kFp4Threads),
                                              0, ctx->stream, pdl, codes, scales, g, rows, cols, (int)(aligned && cols % 8 == 0), out));
    }
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <typename T>
int dequantize_format(shrewq_ctx *ctx, const void *codes, const void *scales, const float *g, size_t rows, size_t cols, bool nv, void *out) {
    const uint32_t *c = static_cast<const uint32_t *>(codes);
    const uint8_t *s = static_cast<const uint8_t *>(scales);
    return nv ? dequantize_as<T, true>(ctx, c, s, g, rows, cols, static_cast<T *>(out)) : dequantize_as<T, false>(ctx, c, s, nullptr, rows, cols, static_cast<T *>(out));
}

}  // namespace

// x: [rows][cols] with a row stride of ld elements.  g (NV): the tensor scale, read, or found and written where find_g is set: the words at g, of
// which those behind the first are workspace
int launch_quantize_fp4(shrewq_ctx *ctx, const void *x, int x_dtype, size_t rows, size_t cols, size_t ld, bool nv, float *g, int find_g,
                        void *codes, void *scales) {
    if (rows * cols == 0) {
        // an empty tensor has no largest value: the scale that a tensor of zeros gets
        if (nv && find_g) return fill_f32(ctx, g, 1.0f);
        return SHREWQ_OK;
    }
    if (x_dtype == SHREWQ_F32) return quantize_format<float>(ctx, x, rows, cols, ld, nv, g, find_g, codes, scales);
    if (x_dtype == SHREWQ_BF16) return quantize_format<__nv_bfloat16>(ctx, x, rows, cols, ld, nv, g, find_g, codes, scales);
    return quantize_format<__half>(ctx, x, rows, cols, ld, nv, g, find_g, codes, scales);
}

int launch_dequantize_fp4(shrewq_ctx *ctx, const void *codes, const void *scales, const float *g, size_t rows, size_t cols, bool nv, int out_dtype, void *out) {
    if (out_dtype == SHREWQ_F32) return dequantize_format<float>(ctx, codes, scales, g, rows, cols, nv, out);
    if (out_dtype == SHREWQ_BF16) return dequantize_format<__nv_bfloat16>(ctx, codes, scales, g, rows, cols, nv, out);
    return dequantize_format<__half>(ctx, codes, scales, g, rows, cols, nv, out);
}

}  // namespace shrewq
