// CPU run of the 4-bit floating point quantizer and dequantizer, of the small-batch forward over such weights and of the norms around a
// block (shrew_b200/csrc/fp4_kernels.cuh, gemv_fp4_kernels.cuh, norm_kernels.cuh) under the CUDA stand-in.  TEST INFRASTRUCTURE
// ONLY; see cuda_shim.h.  dtype: 0 f32, 1 bf16, 2 f16.
#include "cuda_shim_fp4.h"
#include "../../shrew_b200/csrc/gemv_fp4_kernels.cuh"
#include "../../shrew_b200/csrc/norm_kernels.cuh"

using namespace shrewq;

namespace {

template <typename T, bool NV>
void quantize(const void *x, size_t rows, size_t cols, size_t ld, float *g, int find, int route, unsigned grid, void *codes, void *scales) {
    const T *p = static_cast<const T *>(x);
    uint32_t *c = static_cast<uint32_t *>(codes);
    uint8_t *s = static_cast<uint8_t *>(scales);
    const int source = !(NV && find) ? kScaleGiven : (unsigned)find > grid ? (int)grid : kScaleFound;
    if (source != kScaleGiven) {
        if (source == kScaleFound && grid > 1) *g = 0.0f;
        if (route == 0) emu::launch(grid, kFp4Threads, [&] { fp4_tensor_scale_kernel<T, true>(p, rows, cols, ld, g, source > 0); });
        else emu::launch(grid, kFp4Threads, [&] { fp4_tensor_scale_kernel<T, false>(p, rows, cols, ld, g, source > 0); });
    }
    if (route == 0) {
        const size_t groups = rows * cols / 8;
        auto kern = NV && source != kScaleGiven ? fp4_quantize_flat_kernel<T, NV, !NV, 4> : fp4_quantize_flat_kernel<T, NV, true, 4>;
        emu::launch((unsigned)((groups + kFp4Threads * 4 - 1) / (kFp4Threads * 4)), kFp4Threads, [&] { kern(p, groups, g, source, c, s); });
    } else {
        const size_t blocks = (cols + 31) / 32 * (NV ? 2 : 1), threads = (blocks * (NV ? 2 : 4) + 31) / 32 * 32;
        const int vec_ok = (reinterpret_cast<uintptr_t>(p) % (8 * sizeof(T))) == 0 && ld % 8 == 0;
        emu::launch((unsigned)std::min<size_t>(rows, 3), (unsigned)std::min<size_t>(threads, kFp4Threads), [&] {
            fp4_quantize_rows_kernel<T, NV>(p, rows, cols, ld, vec_ok, g, source, blocks, c, s);
        });
    }
}

template <typename T, bool NV>
void dequantize(const void *codes, const void *scales, const float *g, size_t rows, size_t cols, int route, void *out) {
    const uint32_t *c = static_cast<const uint32_t *>(codes);
    const uint8_t *s = static_cast<const uint8_t *>(scales);
    T *o = static_cast<T *>(out);
    const size_t groups = rows * cols / 8;
    if (route == 0)
        emu::launch((unsigned)((groups + kFp4Threads * 4 - 1) / (kFp4Threads * 4)), kFp4Threads, [&] { fp4_dequantize_flat_kernel<T, NV, 4>(c, s, g, groups, o); });
    else
        emu::launch(3, kFp4Threads, [&] { fp4_dequantize_rows_kernel<T, NV>(c, s, g, rows, cols, (reinterpret_cast<uintptr_t>(o) & 31) == 0 && cols % 8 == 0, o); });
}

template <bool NV>
struct Weight {
    std::vector<uint8_t> pieces;
    std::vector<float> alpha;
    Fp4Params params{0.0f, 0.0f, 0, -1};
    Weight(const uint8_t *scales, const float *g, size_t N, size_t K) {
        const size_t n_pieces = (K + 255) / 256 * (NV ? 4 : 2);
        alpha.assign(N, 0.0f);
        pieces.assign((N + 127) / 128 * n_pieces * 512, 0xEE);
        emu::launch(3, 256, [&] { fp4_scale_pieces_kernel<NV>(scales, g, N, (K + 31) / 32 * (NV ? 2 : 1), n_pieces, pieces.data(), &params, 1.0f, alpha.data()); });
    }
};

template <bool NV, bool GATED, typename T>
void forward(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const void *x, int M, int N, int K, float *y,
             size_t ldy, int epilogue, unsigned ctas) {
    const size_t steps = (K + 127) / 128;
    Weight<NV> w0(scales[0], g[0], N, K);
    Weight<NV> w1(scales[GATED ? 1 : 0], g[GATED ? 1 : 0], N, K);
    const Fp4Operand a{codes[0], w0.pieces.data(), &w0.params, bias[0]}, b{codes[GATED ? 1 : 0], w1.pieces.data(), &w1.params, bias[GATED ? 1 : 0]};
    const unsigned tiles = (unsigned)((N + 127) / 128 * (GATED ? 16 : 8));
    const int vec_ok = (reinterpret_cast<uintptr_t>(x) % (8 * sizeof(T))) == 0 && K % 8 == 0;
    emu::launch(tiles < ctas ? tiles : ctas, kGemv4Threads, kGemv4RingBytes + XTerms<T>::kMost * steps * 256 * M,
                [&] { gemv_fp4_kernel<NV, GATED, T, float>(a, b, static_cast<const T *>(x), vec_ok, y, M, N, K, ldy, epilogue); });
}

template <typename TX, typename TB, typename TY>
void norm_typed(const NormArgs &a, int V, unsigned grid) {
    const size_t groups = ((size_t)a.D + 7) / 8;
    switch (V) {
        case 1: emu::launch(grid, 64, [&] { residual_norm_kernel<TX, TB, TY, 1, true>(a); }); break;
        case 4: emu::launch(grid, 32, [&] { residual_norm_kernel<TX, TB, TY, 4, true>(a); }); break;
        default: emu::launch(grid, (unsigned)(((groups + 1) / 2 + 31) / 32 * 32), [&] { residual_norm_kernel<TX, TB, TY, 2, false>(a); });
    }
}

int outcome() { return emu::g_failed.exchange(false) ? -1 : 0; }

}  // namespace

extern "C" long emu_read_only_loads() { return emu::g_read_only_loads.exchange(0); }

// route: 0 = whole aligned rows as one stream, 1 = any rows
extern "C" int emu_fp4_quantize(const void *x, int dtype, size_t rows, size_t cols, size_t ld, int nv, float *g, int find, int route, unsigned grid, void *codes,
                                void *scales) {
#define CALL(T) (nv ? quantize<T, true>(x, rows, cols, ld, g, find, route, grid, codes, scales) : quantize<T, false>(x, rows, cols, ld, g, find, route, grid, codes, scales))
    dtype == 0 ? CALL(float) : dtype == 1 ? CALL(__nv_bfloat16) : CALL(__half);
#undef CALL
    return outcome();
}

extern "C" int emu_fp4_dequantize(const void *codes, const void *scales, const float *g, size_t rows, size_t cols, int nv, int route, int dtype, void *out) {
#define CALL(T) (nv ? dequantize<T, true>(codes, scales, g, rows, cols, route, out) : dequantize<T, false>(codes, scales, g, rows, cols, route, out))
    dtype == 0 ? CALL(float) : dtype == 1 ? CALL(__nv_bfloat16) : CALL(__half);
#undef CALL
    return outcome();
}

extern "C" int emu_fp4_forward(const uint8_t *const *codes, const uint8_t *const *scales, const float *const *g, const float *const *bias, const void *x, int x_f32,
                               int M, int N, int K, int nv, int gated, float *y, size_t ldy, int epilogue, unsigned ctas) {
#define CALL(NV, G)                                                                                              \
    (x_f32 ? forward<NV, G, float>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, ctas)                   \
           : forward<NV, G, __nv_bfloat16>(codes, scales, g, bias, x, M, N, K, y, ldy, epilogue, ctas))
    if (nv) gated ? CALL(true, true) : CALL(true, false);
    else gated ? CALL(false, true) : CALL(false, false);
#undef CALL
    return outcome();
}

extern "C" int emu_residual_norm(const void *x, const void *branch, const void *gate, size_t ldx, size_t ldb, size_t ldg, const float *post_w, const float *post_b,
                                 const float *pre_w, const float *pre_b, void *r, void *h, size_t M, int D, int post, int pre, int gate_kind, float eps,
                                 float residual_scale, float branch_scale, int vec, int x_dtype, int b_dtype, int h_dtype, int V, unsigned grid) {
    const NormArgs a{x, branch, gate, ldx, ldb, ldg, post_w, post_b, pre_w, pre_b, r, h, M, D, post, pre, gate_kind, eps, eps, residual_scale, branch_scale, vec};
    const int which = x_dtype * 4 + b_dtype * 2 + h_dtype;
    switch (which) {
        case 0: norm_typed<float, float, float>(a, V, grid); break;
        case 1: norm_typed<float, float, __nv_bfloat16>(a, V, grid); break;
        case 3: norm_typed<float, __nv_bfloat16, __nv_bfloat16>(a, V, grid); break;
        case 7: norm_typed<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(a, V, grid); break;
        default: return -2;
    }
    return outcome();
}
