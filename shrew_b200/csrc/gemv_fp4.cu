// Launchers of the forward of a few tokens with 4-bit microscaled weights, and of a handle's copy of the scales (device code and its
// description: gemv_fp4_kernels.cuh).
#include <cuda_fp16.h>

#include "gemm_tcgen05_launch.cuh"
#include "gemv_fp4_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

template <bool NV, bool GATED, typename T, typename YT>
int launch_one(shrewq_ctx *ctx, const Fp4Forward &a, size_t staged) {
    const size_t tiles = (a.N + 127) / 128 * (GATED ? 16 : 8);
    const Fp4Operand w0{a.w->codes, a.w->pieces, a.w->params, a.bias};
    const Fp4Operand w1 = GATED ? Fp4Operand{a.up->codes, a.up->pieces, a.up->params, a.bias_up} : w0;
    auto kern = gemv_fp4_kernel<NV, GATED, T, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    int rc = set_smem_attr_once(ctx, kern, kGemv4RingBytes + kGemv4StagedBytes, attr_done);
    if (rc != SHREWQ_OK) return rc;
    const int vec_ok = (reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(T))) == 0 && a.K % 8 == 0;
    SHREWQ_CUDA_TRY(ctx, launch_maybe_pdl(kern, dim3((unsigned)(tiles < (size_t)ctx->sm_count ? tiles : (size_t)ctx->sm_count)), dim3(kGemv4Threads),
                                          kGemv4RingBytes + staged, ctx->stream, a.pdl, w0, w1, static_cast<const T *>(a.x), vec_ok, static_cast<YT *>(a.y), (int)a.M,
                                          (int)a.N, (int)a.K, a.ldy, a.epilogue));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <typename T>
int launch_typed(shrewq_ctx *ctx, const Fp4Forward &a, size_t staged) {
    const bool nv = a.w->nv, f32 = a.y_dtype == SHREWQ_F32;
#define SHREWQ_GEMV4(NV_, G_) return f32 ? launch_one<NV_, G_, T, float>(ctx, a, staged) : launch_one<NV_, G_, T, __nv_bfloat16>(ctx, a, staged)
    if (nv && a.up) SHREWQ_GEMV4(true, true);
    if (nv) SHREWQ_GEMV4(true, false);
    if (a.up) SHREWQ_GEMV4(false, true);
    SHREWQ_GEMV4(false, false);
#undef SHREWQ_GEMV4
}

size_t staged_bytes(const Fp4Forward &a) { return (a.x_dtype == SHREWQ_F32 ? XTerms<float>::kMost : XTerms<__nv_bfloat16>::kMost) * ((a.K + 127) / 128) * 256 * a.M; }

}  // namespace

bool gemv_fp4_supported(const Fp4Forward &a) { return a.M <= (size_t)kGemv4MaxStaged && staged_bytes(a) <= (size_t)kGemv4StagedBytes; }

int launch_gemv_fp4(shrewq_ctx *ctx, const Fp4Forward &a) {
    return a.x_dtype == SHREWQ_F32 ? launch_typed<float>(ctx, a, staged_bytes(a)) : launch_typed<__nv_bfloat16>(ctx, a, staged_bytes(a));
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
