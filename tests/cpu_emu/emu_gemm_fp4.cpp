// CPU run of the 4-bit by 4-bit forward (shrew_b200/csrc/gemm_fp4_kernels.cuh): activations quantized by the quantizer's own device code,
// tensor maps and grid as in the launcher.  TEST INFRASTRUCTURE ONLY; see cuda_shim.h.
#include "cuda_shim_fp4.h"
#include "cuda_shim_tcgen05.h"
#include "cuda_shim_tcgen05_pair.h"
#include "cuda_shim_cluster.h"
#include "cuda_shim_tcgen05_fp4.h"
#include "../../shrew_b200/csrc/gemv_fp4_kernels.cuh"
#include "../../shrew_b200/csrc/gemm_fp4_kernels.cuh"
#include "../../shrew_b200/csrc/gemm_fp4_pair_kernels.cuh"
#include "../../shrew_b200/csrc/gemm_fp4_bf16_kernels.cuh"
#include "../../shrew_b200/csrc/gemm_fp4_f16_kernels.cuh"

using namespace shrewq;

namespace {

uint8_t *aligned(std::vector<uint8_t> &raw, size_t n, uint8_t fill) {
    raw.assign(n + 256, fill);
    return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw.data()) + 255) & ~uintptr_t(255));
}
CUtensorMap map2d(const void *base, uint64_t inner, uint64_t outer, uint32_t box_inner, uint32_t box_outer, uint32_t elem = 1, int swizzle = 128) {
    return CUtensorMap{base, elem, inner, outer, inner * elem, box_inner, box_outer, swizzle};
}

// a grid of tiles, each tile one CTA or (split) a cluster of two
void launch_tiles(size_t tiles, int split, unsigned threads, size_t smem, const std::function<void()> &body) {
    if (split) emu::launch_cluster2((unsigned)tiles * 2, 1, 1, threads, smem, body);
    else emu::launch((unsigned)tiles, threads, smem, body);
}
int outcome(const DeviceStatus &status) { return status.timeout_flag ? -2 : emu::g_failed.exchange(false) ? -1 : 0; }

template <int TOK, bool NV, bool GATED>
int run(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const float *x, float x_scale, int M, int N, int K,
        float *y, size_t ldy, int epilogue, int split) {
    using C = Fp4Cfg<TOK, NV, GATED>;
    const size_t pitch = (K + 31) / 32 * 16, pieces = (size_t)(K + 255) / 256 * C::kPieces;
    std::vector<uint8_t> raw[4];
    std::vector<float> alpha[2];
    uint8_t *wp[2];
    Fp4Params params[2];
    for (int i = 0; i < C::kMats; ++i) {
        wp[i] = aligned(raw[i], (N + 127) / 128 * pieces * 512, 0xEE);
        alpha[i].assign(N, 0.0f);
        params[i] = Fp4Params{0.0f, 0.0f, 0, -1};
        emu::launch(2, 256, [&] {
            fp4_scale_pieces_kernel<NV>(scales[i], g[i], N, (K + 31) / 32 * (NV ? 2 : 1), pieces, wp[i], &params[i], NV ? x_scale : 1.0f, alpha[i].data());
        });
    }
    // (what the quantizer leaves alone is a NaN scale)
    uint8_t *xc = aligned(raw[2], M * pitch, 0xEE), *xp = aligned(raw[3], (M + 127) / 128 * pieces * 512, 0xFF);
    const size_t blocks = pieces * 4, threads = std::min<size_t>(blocks * (NV ? 2 : 4), kFp4Threads);
    emu::launch(M, (unsigned)threads, [&] {
        fp4_quantize_acts_kernel<float, NV>(x, M, K, (reinterpret_cast<uintptr_t>(x) & 31) == 0 && K % 8 == 0, &params[0].x_scale, (K + 255) / 256, reinterpret_cast<uint32_t *>(xc), xp);
    });
    const Operands ops{alpha[0].data(), bias[0], alpha[GATED ? 1 : 0].data(), bias[GATED ? 1 : 0]};
    DeviceStatus status{0, 0, 0, 0};
    if (split == 2) {  // CTA pairs
        const int per = GATED ? 128 : 256, tiles = (N + per - 1) / per * ((M + kPairTok - 1) / kPairTok), pairs = tiles < 2 ? tiles : 2;
        emu::launch_cluster2((unsigned)(2 * pairs), 1, 1, kPairThreads, Fp4PairCfg<NV, GATED, float>::kSmemBytes, [&] {
            gemm_fp4_pair_kernel<NV, GATED, float>(codes[0], codes[GATED ? 1 : 0], xc, wp[0], wp[GATED ? 1 : 0], xp, ops, y, M, N, K, ldy, epilogue, tiles, pairs, &status);
        });
        return outcome(status);
    }
    const int rounds = (K + kFp4StageK - 1) / kFp4StageK, per_cta = split ? (rounds + 1) / 2 : rounds;
    launch_tiles((size_t)(N + 127) / 128 * ((M + TOK - 1) / TOK), split, kFp4GemmThreads, C::kSmemRequest, [&] {
        gemm_fp4_kernel<TOK, NV, GATED, float>(codes[0], codes[GATED ? 1 : 0], xc, wp[0], wp[GATED ? 1 : 0], xp, ops, y, M, N, K, ldy, epilogue, split ? 2 : 1, per_cta, &status);
    });
    return outcome(status);
}

// activations as they come: bf16 straight from x where its rows allow it (XT 1), f32 in three terms
template <int TOK, int XT, bool NV, bool GATED>
int run_w4(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const void *x, int M, int N, int K, float *y,
           size_t ldy, int epilogue, int split) {
    using C = W4Cfg<TOK, XT, NV, GATED>;
    const size_t pitch = (K + 31) / 32 * 16, pieces = (size_t)(K + 255) / 256 * (NV ? 4 : 2), Kp = pitch * 2;
    std::vector<uint8_t> raw[3];
    std::vector<float> alpha[2];
    uint8_t *wp[2];
    Fp4Params params[2];
    for (int i = 0; i < C::kMats; ++i) {
        wp[i] = aligned(raw[i], (N + 127) / 128 * pieces * 512, 0xEE);
        alpha[i].assign(N, 0.0f);
        params[i] = Fp4Params{0.0f, 0.0f, 0, -1};
        emu::launch(2, 256, [&] { fp4_scale_pieces_kernel<NV>(scales[i], g[i], N, (K + 31) / 32 * (NV ? 2 : 1), pieces, wp[i], &params[i], 1.0f, alpha[i].data()); });
    }
    const bool direct = XT == 1 && K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    uint8_t *rows = aligned(raw[2], XT * M * Kp * 2, 0xFF);  // (what is not staged is a NaN)
    if (!direct) {
        uint16_t *t = reinterpret_cast<uint16_t *>(rows);
        if (XT == 3) emu::launch(3, 256, [&] { stage_bf16_kernel<float, XT>(static_cast<const float *>(x), M, K, Kp, 0, t); });
        else emu::launch(3, 256, [&] { stage_bf16_kernel<__nv_bfloat16, XT>(static_cast<const __nv_bfloat16 *>(x), M, K, Kp, 0, t); });
    }
    const int box = GATED ? 64 : 128;
    const CUtensorMap tw = map2d(codes[0], pitch, N, 64, box, 1, 64), tw2 = map2d(codes[GATED ? 1 : 0], pitch, N, 64, box, 1, 64);
    const CUtensorMap tx = map2d(direct ? x : rows, direct ? K : Kp, XT * M, 64, TOK, 2);
    const Operands ops{alpha[0].data(), bias[0], alpha[GATED ? 1 : 0].data(), bias[GATED ? 1 : 0]};
    DeviceStatus status{0, 0, 0, 0};
    const int rounds = (K + kW4StageK - 1) / kW4StageK, per_cta = split ? (rounds + 1) / 2 : rounds;
    launch_tiles((size_t)(N + box - 1) / box * ((M + TOK - 1) / TOK), split, kW4Threads, C::kSmemRequest, [&] {
        gemm_w4_bf16_kernel<TOK, XT, NV, GATED, float>(tw, tw2, tx, wp[0], wp[GATED ? 1 : 0], ops, y, M, N, K, ldy, epilogue, split ? 2 : 1, per_cta, &status);
    });
    return outcome(status);
}

// up to 32 tokens, activations staged as f16 terms
template <int TOK, bool NV, bool GATED, typename T>
int run_h4(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const void *x, int M, int N, int K, float *y,
           size_t ldy, int epilogue, int split) {
    using C = H4Cfg<TOK, NV, GATED>;
    const size_t pitch = (K + 31) / 32 * 16, pieces = (size_t)(K + 255) / 256 * (NV ? 4 : 2), Kp = pitch * 2;
    std::vector<uint8_t> raw[3];
    std::vector<float> alpha[2];
    uint8_t *wp[2];
    Fp4Params params[2];
    for (int i = 0; i < C::kMats; ++i) {
        wp[i] = aligned(raw[i], (N + 127) / 128 * pieces * 512, 0xEE);
        alpha[i].assign(N, 0.0f);
        params[i] = Fp4Params{0.0f, 0.0f, 0, -1};
        emu::launch(2, 256, [&] { fp4_scale_pieces_kernel<NV>(scales[i], g[i], N, (K + 31) / 32 * (NV ? 2 : 1), pieces, wp[i], &params[i], 1.0f, alpha[i].data()); });
    }
    uint8_t *terms = aligned(raw[2], XTerms<T>::kMost * M * Kp * 2, 0x7E);
    std::vector<int> exps(M), counts(M);
    emu::launch(M, (unsigned)(Kp / 8 >= 256 ? 256 : (Kp / 8 + 31) / 32 * 32), [&] {
        stage_f16_kernel<T>(static_cast<const T *>(x), M, K, (int)Kp, (reinterpret_cast<uintptr_t>(x) & 31) == 0 && K % 8 == 0, reinterpret_cast<uint4 *>(terms),
                            exps.data(), counts.data());
    });
    const int box = GATED ? 64 : 128;
    const CUtensorMap tw = map2d(codes[0], pitch, N, 64, box, 1, 64), tw2 = map2d(codes[GATED ? 1 : 0], pitch, N, 64, box, 1, 64);
    const CUtensorMap tx = map2d(terms, Kp, XTerms<T>::kMost * M, 64, TOK, 2);
    const Fp4Operand w0{codes[0], wp[0], &params[0], bias[0]}, w1{codes[GATED ? 1 : 0], wp[GATED ? 1 : 0], &params[GATED ? 1 : 0], bias[GATED ? 1 : 0]};
    DeviceStatus status{0, 0, 0, 0};
    const int rounds = (K + kH4StageK - 1) / kH4StageK, per_cta = split ? (rounds + 1) / 2 : rounds;
    launch_tiles((size_t)(N + box - 1) / box, split, kH4Threads, C::kSmemBytes, [&] {
        gemm_w4_f16_kernel<TOK, NV, GATED, float>(tw, tw2, tx, w0, w1, alpha[0].data(), alpha[GATED ? 1 : 0].data(), exps.data(), counts.data(), XTerms<T>::kMost, XTerms<T>::kOctaves, y, M,
                                                  N, K, ldy, epilogue, split ? 2 : 1, per_cta, &status);
    });
    return outcome(status);
}

}  // namespace

// split: 1 = the k range of a tile over a cluster of two, 2 = CTA pairs (tok is 256 there, 128 in the list of gated ones).  async_seed: 0 = copies and tensor-core work complete at issue, else deferred in an adversarial order
extern "C" int emu_gemm_fp4(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const float *x, float x_scale,
                            int M, int N, int K, int tok, int nv, int gated, float *y, size_t ldy, int epilogue, int split, unsigned async_seed) {
    emu::g_tma_async_seed = async_seed;
    int rc = -3;
#define CALL(T, NV, G) rc = run<T, NV, G>(codes, scales, g, bias, x, x_scale, M, N, K, y, ldy, epilogue, split)
    if (gated) {
        if (tok == 64) { if (nv) CALL(64, true, true); else CALL(64, false, true); }
        if (tok == 128) { if (nv) CALL(128, true, true); else CALL(128, false, true); }
    } else {
        if (tok == 64) { if (nv) CALL(64, true, false); else CALL(64, false, false); }
        if (tok == 128) { if (nv) CALL(128, true, false); else CALL(128, false, false); }
        if (tok == 256) { if (nv) CALL(256, true, false); else CALL(256, false, false); }
    }
#undef CALL
    emu::g_tma_async_seed = 0;
    return rc;
}

extern "C" int emu_gemm_w4_bf16(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const void *x, int x_f32,
                                int M, int N, int K, int tok, int nv, int gated, float *y, size_t ldy, int epilogue, int split, unsigned async_seed) {
    emu::g_tma_async_seed = async_seed;
    int rc = -3;
    if (tok <= 32) {
#define CALL(T, X) rc = nv ? (gated ? run_h4<T, true, true, X>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split)      \
                                    : run_h4<T, true, false, X>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split))    \
                           : (gated ? run_h4<T, false, true, X>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split)     \
                                    : run_h4<T, false, false, X>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split))
        if (tok == 16) { if (x_f32) CALL(16, float); else CALL(16, __nv_bfloat16); }
        if (tok == 32) { if (x_f32) CALL(32, float); else CALL(32, __nv_bfloat16); }
#undef CALL
        emu::g_tma_async_seed = 0;
        return rc;
    }
#define CALL(T, XT) rc = nv ? (gated ? run_w4<T, XT, true, true>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split)      \
                                     : run_w4<T, XT, true, false>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split))    \
                            : (gated ? run_w4<T, XT, false, true>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split)     \
                                     : run_w4<T, XT, false, false>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, split))
    if (x_f32) CALL(64, 3);
    else if (tok == 64) CALL(64, 1);
    else if (tok == 128) CALL(128, 1);
    else if (tok == 256) CALL(256, 1);
#undef CALL
    emu::g_tma_async_seed = 0;
    return rc;
}
