// CPU run of the 4-bit by 4-bit forward (shrew_b200/csrc/gemm_fp4_kernels.cuh): activations quantized by the quantizer's own device code,
// tensor maps and grid as in the launcher.  TEST INFRASTRUCTURE ONLY; see cuda_shim.h.
#include "cuda_shim_fp4.h"
#include "cuda_shim_tcgen05.h"
#include "cuda_shim_tcgen05_fp4.h"
#include "../../shrew_b200/csrc/gemv_fp4_kernels.cuh"
#include "../../shrew_b200/csrc/gemm_fp4_kernels.cuh"

using namespace shrewq;

namespace {

uint8_t *aligned(std::vector<uint8_t> &raw, size_t n, uint8_t fill) {
    raw.assign(n + 256, fill);
    return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw.data()) + 255) & ~uintptr_t(255));
}
CUtensorMap map2d(const void *base, uint64_t inner, uint64_t outer, uint32_t box_inner, uint32_t box_outer) {
    return CUtensorMap{base, 1, inner, outer, inner, box_inner, box_outer, 128};
}

template <int TOK, bool NV, bool GATED>
int run(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const float *x, float x_scale, int M, int N, int K,
        float *y, size_t ldy, int epilogue) {
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
        fp4_quantize_rows_kernel<float, NV, true>(x, M, K, K, 0, &params[0].x_scale, nullptr, 0, nullptr, blocks, reinterpret_cast<uint32_t *>(xc), xp);
    });
    const CUtensorMap tw = map2d(codes[0], pitch, N, 128, 128), tw2 = map2d(codes[GATED ? 1 : 0], pitch, N, 128, 128), tx = map2d(xc, pitch, M, 128, TOK);
    const Operands ops{alpha[0].data(), bias[0], alpha[GATED ? 1 : 0].data(), bias[GATED ? 1 : 0]};
    DeviceStatus status{0, 0, 0, 0};
    emu::launch((unsigned)((N + 127) / 128 * ((M + TOK - 1) / TOK)), kFp4GemmThreads, C::kSmemRequest, [&] {
        gemm_fp4_kernel<TOK, NV, GATED, float>(tw, tw2, tx, wp[0], wp[GATED ? 1 : 0], xp, ops, y, M, N, K, ldy, epilogue, &status);
    });
    if (status.timeout_flag) return -2;
    return emu::g_failed.exchange(false) ? -1 : 0;
}

}  // namespace

// async_seed: 0 = copies and tensor-core work complete at issue, else deferred in an adversarial order
extern "C" int emu_gemm_fp4(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const float *x, float x_scale,
                            int M, int N, int K, int tok, int nv, int gated, float *y, size_t ldy, int epilogue, unsigned async_seed) {
    emu::g_tma_async_seed = async_seed;
    int rc = -3;
#define CALL(T, NV, G) rc = run<T, NV, G>(codes, scales, g, bias, x, x_scale, M, N, K, y, ldy, epilogue)
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
