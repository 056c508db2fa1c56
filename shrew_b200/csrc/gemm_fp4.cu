// Launchers of the 4-bit by 4-bit forward (device code and its description: gemm_fp4_kernels.cuh): the activations are quantized first, by
// a launch of the quantizer that writes their scales in pieces.
#include <cuda_fp16.h>

#include "gemm_tcgen05_launch.cuh"
#include "fp4_kernels.cuh"
#include "gemm_fp4_kernels.cuh"
#include "gemm_fp4_pair_kernels.cuh"
#include "linear_fp4.cuh"

namespace shrewq {
namespace {

template <typename T, bool NV>
cudaError_t quantize_acts(shrewq_ctx *ctx, const Fp4Forward &a, uint32_t *codes, uint8_t *pieces) {
    const uint32_t units = (uint32_t)((a.K + 255) / 256);
    const int vec_ok = (reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(T))) == 0 && a.K % 8 == 0;
    return launch_maybe_pdl(fp4_quantize_acts_kernel<T, NV>, dim3((unsigned)(a.M < 0x7FFFFFFF ? a.M : 0x7FFFFFFF)),
                            dim3(units < kFp4Threads / 32 ? units * 32 : kFp4Threads), 0, ctx->stream, ctx->tuning.pdl != 0, static_cast<const T *>(a.x), a.M,
                            (uint32_t)a.K, vec_ok, (const float *)&a.w->params->x_scale, units, codes, pieces);
}

size_t pair_tiles(const Fp4Forward &a) { return (a.N + (a.up ? 127 : 255)) / (a.up ? 128 : 256) * ((a.M + kPairTok - 1) / kPairTok); }

template <int TOK, bool NV, bool GATED, typename YT>
int launch_one(shrewq_ctx *ctx, const Fp4Forward &a, const void *codes, const uint8_t *pieces) {
    using C = Fp4Cfg<TOK, NV, GATED>;
    auto kern = gemm_fp4_kernel<TOK, NV, GATED, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    int rc;
    if ((rc = set_smem_attr_once(ctx, kern, C::kSmemRequest, attr_done)) != SHREWQ_OK) return rc;
    const size_t tiles = (a.N + 127) / 128 * ((a.M + TOK - 1) / TOK);
    const Operands ops{a.alpha, a.bias, a.alpha_up, a.bias_up};
    int per_cta;
    const int S = split_over_cluster(tiles, (int)((a.K + kFp4StageK - 1) / kFp4StageK), ctx->sm_count, 2, &per_cta);
    if (tiles * S > 0x7FFFFFFF) return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "4-bit forward: more than 2^31 tiles");
    SHREWQ_CUDA_TRY(ctx, launch_cluster(kern, (unsigned)(tiles * S), kFp4GemmThreads, (size_t)C::kSmemRequest, ctx->stream, a.pdl, S, a.w->codes,
                                        GATED ? a.up->codes : a.w->codes, static_cast<const uint8_t *>(codes), (const uint8_t *)a.w->pieces,
                                          (const uint8_t *)(GATED ? a.up->pieces : a.w->pieces), pieces, ops, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy,
                                          a.epilogue, S, per_cta, ctx->dev_status));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <bool NV, bool GATED, typename YT>
int launch_pair(shrewq_ctx *ctx, const Fp4Forward &a, const void *codes, const uint8_t *pieces) {
    using C = Fp4PairCfg<NV, GATED, YT>;
    auto kern = gemm_fp4_pair_kernel<NV, GATED, YT>;
    static std::atomic<unsigned long long> attr_done{0};
    int rc = set_smem_attr_once(ctx, kern, C::kSmemBytes, attr_done);
    if (rc != SHREWQ_OK) return rc;
    const size_t tiles = pair_tiles(a);
    const int pairs = (int)(tiles < (size_t)ctx->sm_count / 2 ? tiles : (size_t)ctx->sm_count / 2);
    if (tiles > 0x3FFFFFFF) return set_err(ctx, SHREWQ_ERR_UNSUPPORTED, "4-bit forward: more than 2^31 tiles");
    const Operands ops{a.alpha, a.bias, a.alpha_up, a.bias_up};
    SHREWQ_CUDA_TRY(ctx, launch_cluster(kern, (unsigned)(2 * pairs), kPairThreads, (size_t)C::kSmemBytes, ctx->stream, a.pdl, 2, a.w->codes,
                                        GATED ? a.up->codes : a.w->codes, static_cast<const uint8_t *>(codes), (const uint8_t *)a.w->pieces,
                                        (const uint8_t *)(GATED ? a.up->pieces : a.w->pieces), pieces, ops, static_cast<YT *>(a.y), (int)a.M, (int)a.N, (int)a.K, a.ldy,
                                        a.epilogue, (int)tiles, pairs, ctx->dev_status));
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

template <bool NV, typename YT>
int launch_tokens(shrewq_ctx *ctx, const Fp4Forward &a, const void *codes, const uint8_t *pieces) {
    // Pairs of CTAs where their tiles of 256 tokens fill half of the machine (4096 x 11008 with 4096 tokens: 114 us against 134 with single CTAs and the same
    // copies, 512 gated tokens 36 against 45); below, single CTAs, which can share a tile's k.
    if (a.M > 128 && pair_tiles(a) * 4 >= (size_t)ctx->sm_count)
        return a.up ? launch_pair<NV, true, YT>(ctx, a, codes, pieces) : launch_pair<NV, false, YT>(ctx, a, codes, pieces);
    if (a.up) return a.M <= 64 ? launch_one<64, NV, true, YT>(ctx, a, codes, pieces) : launch_one<128, NV, true, YT>(ctx, a, codes, pieces);
    if (a.M <= 64) return launch_one<64, NV, false, YT>(ctx, a, codes, pieces);
    if (a.M <= 128) return launch_one<128, NV, false, YT>(ctx, a, codes, pieces);
    return launch_one<256, NV, false, YT>(ctx, a, codes, pieces);
}

}  // namespace

int encode_fp4_tmap(shrewq_ctx *ctx, const uint8_t *codes, size_t n, size_t k, int box_rows, int box_bytes, void *tmap_out) {
    return encode_2d(ctx, static_cast<CUtensorMap *>(tmap_out), CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, (k + 31) / 32 * 16, n, box_bytes, box_rows,
                     box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

int launch_gemm_fp4(shrewq_ctx *ctx, const Fp4Forward &a) {
    const bool nv = a.w->nv;
    const size_t code_bytes = (a.M * ((a.K + 31) / 32 * 16) + 255) / 256 * 256, piece_bytes = (a.M + 127) / 128 * fp4_pieces(a.K, nv) * 512;
    int rc = ensure_xsplit(ctx, code_bytes + piece_bytes);
    if (rc != SHREWQ_OK) return rc;
    uint32_t *codes = static_cast<uint32_t *>(ctx->xsplit);
    uint8_t *pieces = static_cast<uint8_t *>(ctx->xsplit) + code_bytes;
    const bool f32 = a.x_dtype == SHREWQ_F32;
    SHREWQ_CUDA_TRY(ctx, nv ? (f32 ? quantize_acts<float, true>(ctx, a, codes, pieces) : quantize_acts<__nv_bfloat16, true>(ctx, a, codes, pieces))
                            : (f32 ? quantize_acts<float, false>(ctx, a, codes, pieces) : quantize_acts<__nv_bfloat16, false>(ctx, a, codes, pieces)));
    ctx->launches += 1;
    if (a.y_dtype == SHREWQ_F32) return nv ? launch_tokens<true, float>(ctx, a, codes, pieces) : launch_tokens<false, float>(ctx, a, codes, pieces);
    return nv ? launch_tokens<true, __nv_bfloat16>(ctx, a, codes, pieces) : launch_tokens<false, __nv_bfloat16>(ctx, a, codes, pieces);
}

}  // namespace shrewq
