// Launchers of the tensor-core forward with 4-bit weights and activations as they come (device code and its description:
// gemm_fp4_bf16_kernels.cuh).
#include <cuda_fp16.h>

#include "gemm_tcgen05_launch.cuh"
#include "gemm_fp4_bf16_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

// x_rows: the bf16 operand, XT terms of M rows, Kx columns each
template <int TOK, int XT, bool NV, bool GATED, typename YT>
int launch_one(shrewq_ctx *ctx, const Fp4Forward &a, const void *x_rows, size_t Kx) {
    using C = W4Cfg<TOK, XT, NV, GATED>;
    CUtensorMap tx;
    int rc = encode_2d(ctx, &tx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x_rows, Kx, XT * a.M, 64, TOK, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != SHREWQ_OK) return rc;
    auto kern = gemm_w4_bf16_kernel<TOK, XT, NV, GATED, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    if ((rc = set_smem_attr_once(ctx, kern, C::kSmemRequest, attr_done)) != SHREWQ_OK) return rc;
    constexpr size_t kChan = GATED ? 64 : 128;
    const size_t tiles = (a.N + kChan - 1) / kChan * ((a.M + TOK - 1) / TOK);
    int per_cta;
    const int S = split_over_cluster(tiles, (int)((a.K + kW4StageK - 1) / kW4StageK), ctx->sm_count, 4, &per_cta);
    if (tiles * S > 0x7FFFFFFF) return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "4-bit forward: more than 2^31 tiles");
    const CUtensorMap &tw = *static_cast<const CUtensorMap *>(a.w_tmap), &tw2 = GATED ? *static_cast<const CUtensorMap *>(a.up_tmap) : tw;
    const Operands ops{a.alpha, a.bias, a.alpha_up, a.bias_up};
    SHREWQ_CUDA_TRY(ctx, launch_cluster(kern, (unsigned)(tiles * S), kW4Threads, (size_t)C::kSmemRequest, ctx->stream, a.pdl, S, tw, tw2, tx, (const uint8_t *)a.w->pieces,
                                        (const uint8_t *)(GATED ? a.up->pieces : a.w->pieces), ops, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy, a.epilogue, S,
                                        per_cta, ctx->dev_status));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <bool NV, bool GATED, typename YT>
int launch_tokens(shrewq_ctx *ctx, const Fp4Forward &a, const void *x_rows, size_t Kx, bool three) {
    if (three) return launch_one<64, 3, NV, GATED, YT>(ctx, a, x_rows, Kx);
    if (a.M <= 64) return launch_one<64, 1, NV, GATED, YT>(ctx, a, x_rows, Kx);
    if (a.M <= 128) return launch_one<128, 1, NV, GATED, YT>(ctx, a, x_rows, Kx);
    return launch_one<256, 1, NV, GATED, YT>(ctx, a, x_rows, Kx);
}

template <typename T, int XT>
cudaError_t stage(shrewq_ctx *ctx, const Fp4Forward &a, size_t Kp, uint16_t *terms) {
    const size_t want = (a.M * (Kp / 8) + 255) / 256, cap = (size_t)ctx->sm_count * 32;
    const int vec_ok = (reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(T))) == 0 && a.K % 8 == 0;
    return launch_maybe_pdl(stage_bf16_kernel<T, XT>, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, ctx->stream, ctx->tuning.pdl != 0,
                            static_cast<const T *>(a.x), a.M, a.K, Kp, vec_ok, terms);
}

}  // namespace

int launch_gemm_w4_bf16(shrewq_ctx *ctx, const Fp4Forward &a) {
    const bool f32 = a.x_dtype == SHREWQ_F32;
    // the tensor map takes x as it is where its rows are whole 16-byte pieces; else, and for f32, a staged copy
    const bool direct = !f32 && a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    const void *rows = a.x;
    size_t Kx = a.K;
    if (!direct) {
        Kx = (a.K + 31) / 32 * 32;
        int rc = ensure_xsplit(ctx, (f32 ? 3 : 1) * a.M * Kx * 2);
        if (rc != SHREWQ_OK) return rc;
        uint16_t *terms = static_cast<uint16_t *>(ctx->xsplit);
        SHREWQ_CUDA_TRY(ctx, (f32 ? stage<float, 3>(ctx, a, Kx, terms) : stage<__nv_bfloat16, 1>(ctx, a, Kx, terms)));
        ctx->launches += 1;
        rows = terms;
    }
    const bool nv = a.w->nv, gated = a.up != nullptr;
#define SHREWQ_W4(NV_, G_)                                                                   \
    return a.y_dtype == SHREWQ_F32 ? launch_tokens<NV_, G_, float>(ctx, a, rows, Kx, f32)    \
                                   : launch_tokens<NV_, G_, __nv_bfloat16>(ctx, a, rows, Kx, f32)
    if (nv && gated) SHREWQ_W4(true, true);
    if (nv) SHREWQ_W4(true, false);
    if (gated) SHREWQ_W4(false, true);
    SHREWQ_W4(false, false);
#undef SHREWQ_W4
}

}  // namespace shrewq
