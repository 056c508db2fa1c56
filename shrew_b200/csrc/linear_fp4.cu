// C ABI of the 4-bit microscaled operators and of the norms around a block: argument checks, handles, dispatch.
#include <new>

#include "linear_fp4.cuh"

namespace shrewq {
namespace {

int check_format(shrewq_ctx *ctx, int format, const char *who) {
    if (format != SHREWQ_FP4_MX && format != SHREWQ_FP4_NV)
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "%s: format must be SHREWQ_FP4_MX or SHREWQ_FP4_NV", who);
    return SHREWQ_OK;
}

bool storage16or32(int dtype) { return dtype == SHREWQ_F32 || dtype == SHREWQ_BF16 || dtype == SHREWQ_F16; }
bool act_dtype(int dtype) { return dtype == SHREWQ_F32 || dtype == SHREWQ_BF16; }
size_t size_of(int dtype) { return dtype == SHREWQ_F32 ? 4 : 2; }
bool misaligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// rows * cols values at up to 4 bytes, and padded rows, stay within what a size_t and a kernel's index hold
bool sizes_overflow(size_t rows, size_t cols) { return cols > ((size_t)1 << 40) || (cols != 0 && rows > ((size_t)1 << 48) / cols); }

// Up to 32 tokens: the kernel in f16 (two CTAs an SM, a launch to stage the activations) or the one in bf16 (one CTA an SM, bf16 activations as they
// are).  Measured on weights from cold HBM, us in f16 / in bf16:
//   bf16, tiles for one CTA an SM, which may also share their k: bf16 wins (4096 x 4096, 16 tokens: 19.6 / 9.3; 4096 x 11008: 27.2 / 14.6; 8192 x
//     4096 gated: 20.5 / 16.5), but where more than half of the SMs read the same activations of less than 128 KB again and again (11008 x 4096, 8
//     tokens: 18.3 / 18.6; 16384 x 8192, 5 and 8: 28.4 / 39.4, 29.3 / 27.5);
//   bf16, more tiles, which take bf16 another round: f16 wins (11008 x 4096 gated, 8 and 32 tokens: 25.0 / 33.9, 27.0 / 31.5), until the staging and
//     16 tokens an epilogue chunk outweigh short rows (32768 x 512, 8, 16 and 32 tokens: 9.9 / 11.7, 11.6 / 11.6, 15.6 / 11.2; x 1024: 12.2 / 15.7,
//     13.6 / 15.3, 17.4 / 14.9; 50257 x 256, 5 and 12: 14.5 / 16.4, 17.3 / 16.4);
//   f32, three passes in f16, three products of one pass in bf16: bf16 wins (11008 x 4096, 8 tokens: 33.6 / 25.3; gated 55.0 / 49.8), but for activations
//     of less than 128 KB in three terms, as above (5 tokens: 33.1 / 42.1; 32768 x 2048, 8 and 12: 31.8 / 43.4, 32.7 / 30.1).
bool w4_f16_wins(const shrewq_ctx *ctx, const Fp4Forward &a) {
    const size_t tiles = (a.N + (a.up ? 63 : 127)) / (a.up ? 64 : 128), sms = (size_t)ctx->sm_count, few = 128 * 1024;
    if (a.x_dtype == SHREWQ_F32) return tiles > sms / 2 && a.K >= 1024 && a.M * a.K * 6 < few;
    return tiles > sms ? a.M < 8 || a.K >= 64 * a.M : tiles > sms / 2 && a.K >= 4096 && a.M * a.K * 2 < few;
}

}  // namespace

int forward_fp4(shrewq_ctx *ctx, const Fp4Forward &a, const char **kernel) {
    // (the kernels round the tokens up to whole tiles in 32 bits, and f32 ones above 32 stand in three terms one behind the other)
    if (a.M > 0x7FFFFFFFu / (a.M > 32 && !a.w->round_x && a.x_dtype == SHREWQ_F32 ? 3 : 1) - 256)
        return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "4-bit forward: %zu tokens are more than 32-bit indexes hold", a.M);
    if (a.w->round_x) {
        *kernel = "tcgen05-fp4";
        return launch_gemm_fp4(ctx, a);
    }
    if (gemv_fp4_supported(a)) {
        *kernel = "mma-fp4";
        return launch_gemv_fp4(ctx, a);
    }
    if (a.M <= 32 && w4_f16_wins(ctx, a)) {
        *kernel = "tcgen05-w4-f16";
        return launch_gemm_w4_f16(ctx, a);
    }
    *kernel = "tcgen05-w4";
    return launch_gemm_w4_bf16(ctx, a);
}

void destroy_fp4(Fp4Weight *w) {
    if (!w) return;
    if (w->pieces) cudaFree(w->pieces);
    if (w->params) cudaFree(w->params);
    delete w;
}

}  // namespace shrewq

using namespace shrewq;

extern "C" {

int shrewq_quantize_fp4(shrewq_ctx *ctx, const void *w_dev, int w_dtype, size_t rows, size_t cols, size_t ldw, int format, float *tensor_scale_dev,
                        int find_tensor_scale, uint8_t *codes_dev, uint8_t *scales_dev) {
    if (!ctx) return set_err(nullptr, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: ctx is NULL");
    int rc = check_format(ctx, format, "quantize_fp4");
    if (rc != SHREWQ_OK) return rc;
    const bool nv = format == SHREWQ_FP4_NV;
    if (!storage16or32(w_dtype)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: w_dtype must be SHREWQ_F32, SHREWQ_BF16 or SHREWQ_F16");
    if (sizes_overflow(rows, cols)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: rows*cols overflows");
    if (ldw < cols) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: ldw (%zu) smaller than cols (%zu)", ldw, cols);
    if (nv && !tensor_scale_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: SHREWQ_FP4_NV needs tensor_scale_dev");
    if (!nv && tensor_scale_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: SHREWQ_FP4_MX has no tensor scale");
    if (find_tensor_scale < 0) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: find_tensor_scale is 0 or a number of f32");
    if (misaligned(tensor_scale_dev, 4) || misaligned(w_dev, size_of(w_dtype)) || misaligned(codes_dev, 4))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: w_dev aligned to its elements, tensor_scale_dev and codes_dev to 4 bytes");
    if (rows * cols != 0 && (!w_dev || !codes_dev || !scales_dev)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "quantize_fp4: NULL buffer");
    SHREWQ_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    return launch_quantize_fp4(ctx, w_dev, w_dtype, rows, cols, ldw, nv, tensor_scale_dev, find_tensor_scale, codes_dev, scales_dev);
}

int shrewq_dequantize_fp4(shrewq_ctx *ctx, const uint8_t *codes_dev, const uint8_t *scales_dev, const float *tensor_scale_dev, size_t rows, size_t cols,
                          int format, int out_dtype, void *out_dev) {
    if (!ctx) return set_err(nullptr, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: ctx is NULL");
    int rc = check_format(ctx, format, "dequantize_fp4");
    if (rc != SHREWQ_OK) return rc;
    const bool nv = format == SHREWQ_FP4_NV;
    if (!storage16or32(out_dtype)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: out_dtype must be SHREWQ_F32, SHREWQ_BF16 or SHREWQ_F16");
    if (sizes_overflow(rows, cols)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: rows*cols overflows");
    if (nv && !tensor_scale_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: SHREWQ_FP4_NV needs tensor_scale_dev");
    if (!nv && tensor_scale_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: SHREWQ_FP4_MX has no tensor scale");
    if (misaligned(tensor_scale_dev, 4) || misaligned(out_dev, size_of(out_dtype)) || misaligned(codes_dev, 4))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: out_dev aligned to its elements, tensor_scale_dev and codes_dev to 4 bytes");
    if (rows * cols == 0) return SHREWQ_OK;
    if (!codes_dev || !scales_dev || !out_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "dequantize_fp4: NULL buffer");
    SHREWQ_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    return launch_dequantize_fp4(ctx, codes_dev, scales_dev, tensor_scale_dev, rows, cols, nv, out_dtype, out_dev);
}

int shrewq_linear_create_fp4(shrewq_ctx *ctx, const uint8_t *codes_dev, const uint8_t *scales_dev, const float *tensor_scale_dev, const float *bias_dev,
                             size_t out_features, size_t in_features, int format, int quantize_activations, float activation_scale, shrewq_linear **out) {
    if (!ctx) return set_err(nullptr, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: ctx is NULL");
    if (!out) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: out is NULL");
    *out = nullptr;
    int rc = check_format(ctx, format, "linear_create_fp4");
    if (rc != SHREWQ_OK) return rc;
    const bool nv = format == SHREWQ_FP4_NV;
    if (!codes_dev || !scales_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: codes_dev / scales_dev is NULL");
    if (out_features == 0 || in_features == 0) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: empty layer");
    if (out_features > 0x7FFFFF00u || in_features > 0x7FFFFF00u)
        return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "linear_create_fp4: dimensions above 2^31");
    if (nv != (tensor_scale_dev != nullptr))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, nv ? "linear_create_fp4: SHREWQ_FP4_NV needs tensor_scale_dev" : "linear_create_fp4: SHREWQ_FP4_MX has no tensor scale");
    if (misaligned(codes_dev, 16) || misaligned(tensor_scale_dev, 4) || misaligned(bias_dev, 4))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: codes_dev must be 16-byte, bias_dev and tensor_scale_dev 4-byte aligned");
    if (quantize_activations && nv && !(activation_scale >= 1e-30f && activation_scale <= 1e30f))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "linear_create_fp4: activation_scale must be a positive number (1e-30 .. 1e30)");
    SHREWQ_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    shrewq_linear *lin = new (std::nothrow) shrewq_linear();
    Fp4Weight *w = new (std::nothrow) Fp4Weight();
    if (!lin || !w) {
        delete lin;
        delete w;
        return set_err(ctx, SHREWQ_ERR_ALLOC, "out of host memory");
    }
    lin->ctx = ctx;
    lin->bias = bias_dev;
    lin->n = out_features;
    lin->k = in_features;
    lin->fp4 = w;
    w->codes = codes_dev;
    w->nv = nv;
    w->round_x = quantize_activations != 0;
    w->x_scale = nv && w->round_x ? activation_scale : 1.0f;  // (activations as they come have none)
    const size_t pieces = fp4_pieces(in_features, nv), bytes = (out_features + 127) / 128 * pieces * 512;
    if (cudaMalloc(&w->pieces, bytes) != cudaSuccess || cudaMalloc(&w->params, sizeof(Fp4Params)) != cudaSuccess ||
        cudaMalloc(&lin->scales_f32, out_features * sizeof(float)) != cudaSuccess) {
        cudaGetLastError();
        shrewq_linear_destroy(lin);
        return set_err(ctx, SHREWQ_ERR_ALLOC, "linear_create_fp4: allocation of %zu bytes for the scales failed", bytes);
    }
    rc = launch_fp4_scale_pieces(ctx, scales_dev, tensor_scale_dev, out_features, (in_features + 31) / 32 * (nv ? 2 : 1), pieces, nv, w->pieces, w->params, w->x_scale,
                                 lin->scales_f32);
    // boxes of the tensor-core kernels that take activations as they come: 128 codes of 128 and, gated, 64 rows
    if (rc == SHREWQ_OK && !w->round_x) rc = encode_fp4_tmap(ctx, codes_dev, out_features, in_features, 128, 64, lin->w_tmap);
    if (rc == SHREWQ_OK && !w->round_x) rc = encode_fp4_tmap(ctx, codes_dev, out_features, in_features, 64, 64, lin->w_tmap64);
    if (rc != SHREWQ_OK) {
        shrewq_linear_destroy(lin);
        return rc;
    }
    *out = lin;
    return SHREWQ_OK;
}

int shrewq_residual_norm(shrewq_ctx *ctx, const shrewq_residual_norm_args *p) {
    if (!ctx) return set_err(nullptr, SHREWQ_ERR_INVALID_ARG, "residual_norm: ctx is NULL");
    if (!p) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: args is NULL");
    if (p->D == 0) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: D is 0");
    if (p->D > 32768) return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "residual_norm: rows of more than 32768 values");
    if (!act_dtype(p->x_dtype) || (p->branch_dev && !act_dtype(p->branch_dtype)) || (p->normed_dev && !act_dtype(p->normed_dtype)))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: types are SHREWQ_F32 and SHREWQ_BF16");
    const auto kind_ok = [](int k) { return k >= SHREWQ_NORM_NONE && k <= SHREWQ_NORM_LAYER; };
    if (!kind_ok(p->post_norm) || !kind_ok(p->pre_norm) || p->gate_kind < SHREWQ_GATE_NONE || p->gate_kind > SHREWQ_GATE_FULL)
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: unknown norm or gate kind");
    if (!p->residual_dev && !p->normed_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: no output");
    if ((p->normed_dev != nullptr) != (p->pre_norm != SHREWQ_NORM_NONE))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: normed_dev goes with a pre_norm");
    if (!p->branch_dev && (p->post_norm != SHREWQ_NORM_NONE || p->gate_kind != SHREWQ_GATE_NONE))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: post_norm and gate need a branch");
    if ((p->gate_dev != nullptr) != (p->gate_kind != SHREWQ_GATE_NONE)) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: gate_dev goes with a gate_kind");
    if ((p->post_norm != SHREWQ_NORM_NONE && !(p->post_eps >= 0.0f)) || (p->pre_norm != SHREWQ_NORM_NONE && !(p->pre_eps >= 0.0f)))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: eps must not be negative");
    if (p->M == 0) return SHREWQ_OK;
    if (!p->x_dev) return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: x_dev is NULL");
    if (p->M > 1 && (p->ldx < p->D || (p->branch_dev && p->ldb < p->D) || (p->gate_kind == SHREWQ_GATE_FULL && p->ldg < p->D)))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: a row stride is smaller than D");
    if (misaligned(p->x_dev, size_of(p->x_dtype)) || (p->branch_dev && (misaligned(p->branch_dev, size_of(p->branch_dtype)) || misaligned(p->gate_dev, size_of(p->branch_dtype)))) ||
        misaligned(p->residual_dev, size_of(p->x_dtype)) || (p->normed_dev && misaligned(p->normed_dev, size_of(p->normed_dtype))) || misaligned(p->post_weight_dev, 4) ||
        misaligned(p->post_bias_dev, 4) || misaligned(p->pre_weight_dev, 4) || misaligned(p->pre_bias_dev, 4))
        return set_err(ctx, SHREWQ_ERR_INVALID_ARG, "residual_norm: a buffer is not aligned to its elements");
    SHREWQ_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    return launch_residual_norm(ctx, p);
}

}  // extern "C"
