// Launchers of the small-batch forward with 4-bit microscaled weights, and of a handle's copy of the scales (device code and its
// description: gemv_fp4_kernels.cuh).
#include <cuda_fp16.h>

#include "gemm_tcgen05_launch.cuh"
#include "gemv_fp4_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

template <int NT, bool NV, bool GATED, bool XS, typename T, typename YT>
int launch_one(shrewq_ctx *ctx, const Fp4Forward &a, const Gemv4X<T> &x, size_t staged) {
    const size_t tiles = (a.N + 127) / 128 * (GATED ? 16 : 8), smem = kGemv4RingBytes + staged;
    const Fp4Operand w0{a.w->codes, a.w->pieces, a.w->params, a.bias};
    const Fp4Operand w1 = GATED ? Fp4Operand{a.up->codes, a.up->pieces, a.up->params, a.bias_up} : w0;
    auto kern = gemv_fp4_kernel<NT, NV, GATED, XS, T, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    int rc = set_smem_attr_once(ctx, kern, kGemv4RingBytes + (XS ? kGemv4StagedBytes : 0), attr_done);
    if (rc != SHREWQ_OK) return rc;
    SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(kern, dim3((unsigned)(tiles < (size_t)ctx->sm_count ? tiles : (size_t)ctx->sm_count)), dim3(kGemv4Threads), smem, ctx->stream,
                                          a.pdl, w0, w1, x, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy, a.epilogue));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <int NT, bool XS, typename T>
int launch_weights(shrewq_ctx *ctx, const Fp4Forward &a, const Gemv4X<T> &x, size_t staged) {
    const bool nv = a.w->nv, f32 = a.y_dtype == SHREWQ_F32;
#define SHREWQ_GEMV4(NV_, G_)                                                                 \
    return f32 ? launch_one<NT, NV_, G_, XS, T, float>(ctx, a, x, staged) : launch_one<NT, NV_, G_, XS, T, __nv_bfloat16>(ctx, a, x, staged)
    if (nv && a.up) SHREWQ_GEMV4(true, true);
    if (nv) SHREWQ_GEMV4(true, false);
    if (a.up) SHREWQ_GEMV4(false, true);
    SHREWQ_GEMV4(false, false);
#undef SHREWQ_GEMV4
}

template <typename T>
int launch_typed(shrewq_ctx *ctx, const Fp4Forward &a) {
    const size_t steps = (a.K + 127) / 128;
    Gemv4X<T> x{static_cast<const T *>(a.x), (reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(T))) == 0 && a.K % 8 == 0, nullptr, nullptr, nullptr};
    // a few tokens are staged by the CTAs themselves: one launch, no workspace
    const size_t staged = XTerms<T>::kMost * steps * 256 * a.M;
    if (a.M <= (size_t)kGemv4MaxStaged && staged <= (size_t)kGemv4StagedBytes) return launch_weights<1, true, T>(ctx, a, x, staged);
    const int NT = a.M <= 8 ? 1 : a.M <= 16 ? 2 : 4;
    const size_t plane = (size_t)NT * steps * 2048;
    int rc = ensure_xsplit(ctx, XTerms<T>::kMost * plane + 2 * a.M * sizeof(int));
    if (rc != SHREWQ_OK) return rc;
    char *base = static_cast<char *>(ctx->xsplit);
    int *exps = reinterpret_cast<int *>(base + XTerms<T>::kMost * plane), *counts = exps + a.M;
    SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(stage_f16_kernel<T>, dim3((unsigned)(8 * NT)), dim3((unsigned)(steps >= 16 ? 256 : (steps * 16 + 31) / 32 * 32)), 0, ctx->stream,
                                          ctx->tuning.pdl != 0, x.x, (int)a.M, (int)a.K, x.vec_ok, reinterpret_cast<uint4 *>(base), exps, counts));
    ctx->launches += 1;
    x.terms = reinterpret_cast<const uint4 *>(base);
    x.exps = exps;
    x.counts = counts;
    if (NT == 1) return launch_weights<1, false, T>(ctx, a, x, 0);
    if (NT == 2) return launch_weights<2, false, T>(ctx, a, x, 0);
    return launch_weights<4, false, T>(ctx, a, x, 0);
}

}  // namespace

int launch_gemv_fp4(shrewq_ctx *ctx, const Fp4Forward &a) {
    return a.x_dtype == SHREWQ_F32 ? launch_typed<float>(ctx, a) : launch_typed<__nv_bfloat16>(ctx, a);
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
