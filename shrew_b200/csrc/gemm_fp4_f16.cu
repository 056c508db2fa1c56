// Launchers of the forward of up to 32 tokens with 4-bit weights in f16 (device code and its description: gemm_fp4_f16_kernels.cuh).
#include <cuda_fp16.h>

#include "gemm_tcgen05_launch.cuh"
#include "gemm_fp4_f16_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

struct Staged {
    const void *terms;
    const int *exps, *counts;
    int most, octaves;
};

template <int TOK, bool NV, bool GATED, typename YT>
int launch_one(shrewq_ctx *ctx, const Fp4Forward &a, const Staged &x) {
    using C = H4Cfg<TOK, NV, GATED>;
    CUtensorMap tx;
    // (f16 and bf16 are the same to a copy)
    int rc = encode_2d(ctx, &tx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x.terms, (a.K + 31) / 32 * 32, x.most * a.M, 64, TOK, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != SHREWQ_OK) return rc;
    auto kern = gemm_w4_f16_kernel<TOK, NV, GATED, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    if ((rc = set_smem_attr_once(ctx, kern, C::kSmemRequest, attr_done)) != SHREWQ_OK) return rc;
    const size_t tiles = (a.N + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
    int per_cta;
    const int S = split_over_cluster(tiles, (int)((a.K + kH4StageK - 1) / kH4StageK), 2 * ctx->sm_count, 4, &per_cta);
    if (tiles * S > 0x7FFFFFFF) return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "4-bit forward: more than 2^31 tiles");
    const CUtensorMap &tw = *static_cast<const CUtensorMap *>(a.w_tmap), &tw2 = GATED ? *static_cast<const CUtensorMap *>(a.up_tmap) : tw;
    const Fp4Operand w0{a.w->codes, a.w->pieces, a.w->params, a.bias};
    const Fp4Operand w1 = GATED ? Fp4Operand{a.up->codes, a.up->pieces, a.up->params, a.bias_up} : w0;
    SHREWQ_CUDA_TRY(ctx, launch_cluster(kern, (unsigned)(tiles * S), kH4Threads, (size_t)C::kSmemRequest, ctx->stream, a.pdl, S, tw, tw2, tx, w0, w1, a.alpha,
                                        GATED ? a.alpha_up : a.alpha, (const int *)x.exps, (const int *)x.counts, x.most, x.octaves, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy,
                                        a.epilogue, S, per_cta, ctx->dev_status));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <bool NV, bool GATED, typename YT>
int launch_tokens(shrewq_ctx *ctx, const Fp4Forward &a, const Staged &x) {
    return a.M <= 16 ? launch_one<16, NV, GATED, YT>(ctx, a, x) : launch_one<32, NV, GATED, YT>(ctx, a, x);
}

template <typename T>
cudaError_t stage(shrewq_ctx *ctx, const Fp4Forward &a, size_t Kp, void *terms, int *exps, int *counts) {
    const int vec_ok = (reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(T))) == 0 && a.K % 8 == 0;
    return launch_maybe_pdl(stage_f16_kernel<T>, dim3((unsigned)a.M), dim3((unsigned)(Kp / 8 >= 256 ? 256 : (Kp / 8 + 31) / 32 * 32)), 0, ctx->stream,
                            ctx->tuning.pdl != 0, static_cast<const T *>(a.x), (int)a.M, (int)a.K, (int)Kp, vec_ok, static_cast<uint4 *>(terms), exps, counts);
}

}  // namespace

// M <= 32
int launch_gemm_w4_f16(shrewq_ctx *ctx, const Fp4Forward &a) {
    const bool f32 = a.x_dtype == SHREWQ_F32;
    const size_t Kp = (a.K + 31) / 32 * 32, most = f32 ? XTerms<float>::kMost : XTerms<__nv_bfloat16>::kMost, bytes = (most * a.M * Kp * 2 + 255) / 256 * 256;
    int rc = ensure_xsplit(ctx, bytes + 2 * a.M * sizeof(int));
    if (rc != SHREWQ_OK) return rc;
    int *exps = reinterpret_cast<int *>(static_cast<char *>(ctx->xsplit) + bytes), *counts = exps + a.M;
    SHREWQ_CUDA_TRY(ctx, (f32 ? stage<float>(ctx, a, Kp, ctx->xsplit, exps, counts) : stage<__nv_bfloat16>(ctx, a, Kp, ctx->xsplit, exps, counts)));
    ctx->launches += 1;
    const Staged x{ctx->xsplit, exps, counts, (int)most, f32 ? XTerms<float>::kOctaves : XTerms<__nv_bfloat16>::kOctaves};
    const bool nv = a.w->nv;
#define SHREWQ_H4(NV_, G_) return a.y_dtype == SHREWQ_F32 ? launch_tokens<NV_, G_, float>(ctx, a, x) : launch_tokens<NV_, G_, __nv_bfloat16>(ctx, a, x)
    if (nv && a.up) SHREWQ_H4(true, true);
    if (nv) SHREWQ_H4(true, false);
    if (a.up) SHREWQ_H4(false, true);
    SHREWQ_H4(false, false);
#undef SHREWQ_H4
}

}  // namespace shrewq
