// Launchers of the small-batch forward with 4-bit microscaled weights, and of a handle's copy of the scales (device code and its
// description: gemv_fp4_kernels.cuh).
#include <cuda_fp16.h>

#include "common.cuh"
#include "gemv_fp4_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

template <int NT, int RT, bool NV, bool GATED, typename YT>
cudaError_t launch_one(shrewq_ctx *ctx, const Fp4Forward &a, const uint16_t *terms, const int *exps, const int *counts) {
    const size_t tiles = (a.N + 127) / 128 * (GATED ? 16 : 8);
    const Fp4Operand w0{a.w->codes, a.w->pieces, a.w->params, a.bias};
    const Fp4Operand w1 = GATED ? Fp4Operand{a.up->codes, a.up->pieces, a.up->params, a.bias_up} : w0;
    return launch_maybe_pdl(gemv_fp4_kernel<NT, RT, NV, GATED, YT>, dim3((unsigned)((tiles + RT - 1) / RT)), dim3(kGemv4Warps * 32), 0, ctx->stream, a.pdl, w0,
                            w1, terms, exps, counts, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy, a.epilogue);
}

template <bool NV, bool GATED, typename YT>
cudaError_t launch_tokens(shrewq_ctx *ctx, const Fp4Forward &a, const uint16_t *terms, const int *exps, const int *counts) {
    if (a.M <= 8) return launch_one<1, 1, NV, GATED, YT>(ctx, a, terms, exps, counts);
    if (a.M <= 16) return launch_one<2, 1, NV, GATED, YT>(ctx, a, terms, exps, counts);
    return launch_one<4, 1, NV, GATED, YT>(ctx, a, terms, exps, counts);
}

}  // namespace

int launch_gemv_fp4(shrewq_ctx *ctx, const Fp4Forward &a) {
    const size_t Kp = (a.K + 31) / 32 * 32, plane = a.M * Kp * sizeof(uint16_t);
    int rc = ensure_xsplit(ctx, 3 * plane + 2 * a.M * sizeof(int));
    if (rc != SHREWQ_OK) return rc;
    char *base = static_cast<char *>(ctx->xsplit);
    uint16_t *terms = reinterpret_cast<uint16_t *>(base);
    int *exps = reinterpret_cast<int *>(base + 3 * plane), *counts = exps + a.M;
    const bool pdl = ctx->tuning.pdl != 0;
    const unsigned threads = (unsigned)(Kp / 8 >= 256 ? 256 : (Kp / 8 + 31) / 32 * 32);
    const size_t esz = a.x_dtype == SHREWQ_F32 ? 4 : 2;
    const int vec_ok = (reinterpret_cast<uintptr_t>(a.x) % (8 * esz)) == 0 && a.K % 8 == 0;
    if (a.x_dtype == SHREWQ_F32)
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(stage_f16_kernel<float>, dim3((unsigned)a.M), dim3(threads), 0, ctx->stream, pdl, static_cast<const float *>(a.x),
                                              (int)a.M, (int)a.K, (int)Kp, vec_ok, terms, exps, counts));
    else
        SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(stage_f16_kernel<__nv_bfloat16>, dim3((unsigned)a.M), dim3(threads), 0, ctx->stream, pdl,
                                              static_cast<const __nv_bfloat16 *>(a.x), (int)a.M, (int)a.K, (int)Kp, vec_ok, terms, exps, counts));
    cudaError_t e;
    const bool nv = a.w->nv, gated = a.up != nullptr, f32 = a.y_dtype == SHREWQ_F32;
#define SHREWQ_GEMV4(NV_, G_)                                                                      \
    e = f32 ? launch_tokens<NV_, G_, float>(ctx, a, terms, exps, counts) : launch_tokens<NV_, G_, __nv_bfloat16>(ctx, a, terms, exps, counts)
    if (nv && gated) SHREWQ_GEMV4(true, true);
    else if (nv) SHREWQ_GEMV4(true, false);
    else if (gated) SHREWQ_GEMV4(false, true);
    else SHREWQ_GEMV4(false, false);
#undef SHREWQ_GEMV4
    SHREWQ_CUDA_TRY(ctx, e);
    ctx->launches += 2;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

int launch_fp4_scale_pieces(shrewq_ctx *ctx, const uint8_t *scales, const float *g, size_t N, size_t blocks, size_t pieces, bool nv, uint8_t *out,
                            Fp4Params *params, float x_scale, float *alpha) {
    SHREWQ_CUDA_TRY(ctx, cudaMemsetAsync(&params->max_byte, 0, sizeof(int), ctx->stream));
    SHREWQ_CUDA_TRY(ctx, cudaMemsetAsync(&params->min_byte, 0xFF, sizeof(int), ctx->stream));
    const size_t words = (N + 127) / 128 * 128 * pieces, want = (words + 255) / 256, cap = (size_t)ctx->sm_count * 16;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    if (nv) fp4_scale_pieces_kernel<true><<<grid, 256, 0, ctx->stream>>>(scales, g, N, blocks, pieces, out, params, x_scale, alpha);
    else fp4_scale_pieces_kernel<false><<<grid, 256, 0, ctx->stream>>>(scales, g, N, blocks, pieces, out, params, x_scale, alpha);
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

}  // namespace shrewq
