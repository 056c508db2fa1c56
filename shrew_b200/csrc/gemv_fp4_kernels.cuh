// Forward of a layer with 4-bit microscaled weights for up to 32 tokens, sm_100a: warp-level MMA on f16 operands.
//
//   y[m,n] = alpha * sum_k w[n,k] x[m,k] + bias[n],   w = code * block scale  (alpha: the tensor scale of NV, 1 for MX)
//
// Bound by the weight stream (0.53 or 0.56 bytes a weight, read once) and, right behind it, by the widening of the codes: at the
// stream's rate an SM has to widen 46 codes a cycle, so what counts is instructions per code on the 16-lane ALU pipe.  E2M1 -> f16 is
// one conversion for two codes, half as many ALU cycles as any way to bf16 (shifts and masks to move sign, exponent and mantissa),
// and the block scale costs one packed multiplication on the FMA pipe.  Both are exact in f16:
//   NV: code * E4M3 scale has 6 significant bits between 2^-10 and 2688;
//   MX: code * 2^d is exact for d in [-14, 13], so the scales of a tensor are taken in windows of 28 octaves below the largest one; a
//       tensor whose scales span more (the handle knows their range) takes a pass over its codes for every window.
// Activations are f16 too: a pass before this kernel (stage_f16_kernel) scales every token by a power of two to [2^14, 2^15) and writes
// f16 terms: bf16 values down to 2^-32 of their token's largest are exact in the first; where a token has smaller ones a second term
// holds what the first left, times 2^32.  f32 values take three terms of 11 bits each.  The kernel passes over the codes once for every
// term that any token needs, and adds the passes' sums with their weights in f32.  Products are exact, sums are f32.
//
// Mapping.  A CTA of 8 warps takes RT tiles of 16 rows (GATED: 8 gate rows and the 8 up rows of the same channels); the warps deal the
// k range in steps of 128 codes.  mma.sync.m16n8k16 with the weights as the A operand: lane (g = lane / 4, t = lane % 4) loads 16
// bytes = 32 consecutive codes (one MX block, two NV blocks: the scale is the lane's own) of rows g and g + 8 and the 32 activations
// of the same k for token g; MMA step i uses the codes 4i .. 4i+3 of that run for A and B alike.  Four steps are requested at a time, the
// next four before these are used, so that 16 warps keep 64 KB of codes in flight on an SM.  The rows of a tile are 4 neighbours each
// from the 4 groups of 32 that share 16 bytes of scales in the handle's copy (scale_piece_offset), so that scale sectors are used whole.
// The warps' sums meet in shared memory in a fixed order.
//
// Programmatic dependent launch: the first codes and scales are requested before the wait for the previous kernel.
//
// Device code only (PTX behind ptx_fp4.cuh and ptx_small.cuh): also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "../../include/shrewq.h"
#include "fp4_kernels.cuh"
#include "fp4_params.cuh"
#include "ptx_fp4.cuh"
#include "ptx_small.cuh"

namespace shrewq {
namespace {

constexpr int kGemv4Warps = 8;
constexpr int kMxWindow = 28;  // octaves of MX scales that one pass takes

// What the kernels need of one weight matrix (device pointers; params and pieces belong to the handle)
struct Fp4Operand {
    const uint8_t *codes;    // [N][pitch]
    const uint8_t *pieces;   // scales in the order of scale_piece_offset
    const Fp4Params *params;
    const float *bias;
};

// ---- activations -> f16 terms -----------------------------------------------------------------------------------------------
// A CTA a token.  terms: [3][M][Kp] f16 (Kp = K to whole 32s, zeros beyond K); exps[m]: the power of two that the token was divided
// by; counts[m]: terms in use.  Infinities and NaNs stay what they are in the first term and are 0 in the others.
template <typename T>
__global__ void __launch_bounds__(256)
stage_f16_kernel(const T *__restrict__ x, int M, int K, int Kp, int vec_ok, uint16_t *__restrict__ terms, int *__restrict__ exps,
                 int *__restrict__ counts) {
    pdl_launch_dependents();
    __shared__ unsigned int s_max[8], s_more[8];
    pdl_wait();
    const int m = blockIdx.x, threads = (int)blockDim.x, warps = threads >> 5;
    const T *row = x + (size_t)m * K;
    const int groups = Kp >> 3;
    unsigned int top = 0;  // largest exponent field of a finite value
    for (int i = threadIdx.x; i < groups; i += threads) {
        float v[8];
        if (vec_ok && i * 8 + 8 <= K) load_vec8<T>(row + i * 8, v);
        else load_guarded8<T>(row + i * 8, i * 8 < K ? (size_t)(K - i * 8) : 0, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned int e = (__float_as_uint(v[j]) >> 23) & 0xFFu;
            top = e < 255u && e > top ? e : top;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned int other = __shfl_xor_sync(0xFFFFFFFFu, top, o);
        top = other > top ? other : top;
    }
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = s_max[w] > top ? s_max[w] : top;
    // x * 2^(14 - (top - 127)), in two factors that are both ordinary numbers
    const int up = 141 - (int)top;                       // -113 .. 141
    const float f0 = __uint_as_float((uint32_t)(127 + (up > 100 ? 100 : up)) << 23), f1 = __uint_as_float((uint32_t)(127 + (up > 100 ? up - 100 : 0)) << 23);
    constexpr bool kWide = sizeof(T) == 4;               // f32: three terms, 11 octaves apart; bf16: two, 32 apart
    const float next = kWide ? 2048.0f : 4294967296.0f;
    const size_t plane = (size_t)M * Kp;
    unsigned int more = 0;
    for (int i = threadIdx.x; i < groups; i += threads) {
        float v[8];
        if (vec_ok && i * 8 + 8 <= K) load_vec8<T>(row + i * 8, v);
        else load_guarded8<T>(row + i * 8, i * 8 < K ? (size_t)(K - i * 8) : 0, v);
        uint32_t t0[4], t1[4], t2[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = v[2 * j] * f0 * f1, b = v[2 * j + 1] * f0 * f1, ha, hb;
            const auto rest = [&](float &r, float h) {  // what a term left, for the next one
                r = (h - h == 0.0f) ? (r - h) * next : 0.0f;
            };
            t0[j] = pack_f16x2_rn(b, a);
            f32x2_of_f16x2(t0[j], ha, hb);
            rest(a, ha);
            rest(b, hb);
            more |= (a != 0.0f || b != 0.0f) ? 1u : 0u;
            t1[j] = pack_f16x2_rn(b, a);
            if constexpr (kWide) {
                f32x2_of_f16x2(t1[j], ha, hb);
                rest(a, ha);
                rest(b, hb);
                t2[j] = pack_f16x2_rn(b, a);
            } else {
                t2[j] = 0;
            }
        }
        uint16_t *dst = terms + (size_t)m * Kp + i * 8;
        *reinterpret_cast<uint4 *>(dst) = make_uint4(t0[0], t0[1], t0[2], t0[3]);
        *reinterpret_cast<uint4 *>(dst + plane) = make_uint4(t1[0], t1[1], t1[2], t1[3]);
        if constexpr (kWide) *reinterpret_cast<uint4 *>(dst + 2 * plane) = make_uint4(t2[0], t2[1], t2[2], t2[3]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) more |= __shfl_xor_sync(0xFFFFFFFFu, more, o);
    if ((threadIdx.x & 31) == 0) s_more[threadIdx.x >> 5] = more;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 0; w < warps; ++w) more |= s_more[w];
        exps[m] = -up;
        counts[m] = more ? (kWide ? 3 : 2) : 1;
    }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------
// MX: `word` holds the scale bytes of the row's 4 blocks of this step, t the lane's; first: the byte that stands for 2^-14 in this pass
__device__ __forceinline__ uint32_t mx_scale_f16x2(uint32_t word, int t, int first) {
    const uint32_t byte = (word >> (8 * t)) & 0xFFu;
    const uint32_t d = byte - (uint32_t)first;           // 0 .. 27 inside the window
    uint32_t h = d < (uint32_t)kMxWindow ? (d + 1u) << 10 : 0u;
    h = byte == 255u ? 0x7E00u : h;                      // NaN in every pass
    return h * 0x10001u;
}
__device__ __forceinline__ uint32_t dup_lo(uint32_t h) { return __byte_perm(h, h, 0x1010); }
__device__ __forceinline__ uint32_t dup_hi(uint32_t h) { return __byte_perm(h, h, 0x3232); }

template <typename YT>
__device__ __forceinline__ void store_out(YT *p, float v);
template <>
__device__ __forceinline__ void store_out<float>(float *p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store_out<__nv_bfloat16>(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Row of the matrix behind row i of tile `tile`: plain 4 neighbours of each group of 32 (16 rows), gated 2 of each (8 rows)
template <bool GATED>
__device__ __forceinline__ int gemv4_row(int tile, int i) {
    constexpr int kShift = GATED ? 1 : 2, kTiles = 32 >> kShift;  // tiles in 128 rows: 16 gated, 8 plain
    return (tile / kTiles) * 128 + (tile % kTiles) * (1 << kShift) + (i & ((1 << kShift) - 1)) + 32 * (i >> kShift);
}

// NT: token groups of 8 (M <= 8 * NT); RT: tiles of 16 rows a CTA
template <int NT, int RT, bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kGemv4Warps * 32, 2)
gemv_fp4_kernel(Fp4Operand w0, Fp4Operand w1, const uint16_t *__restrict__ terms, const int *__restrict__ exps, const int *__restrict__ counts,
                YT *__restrict__ y, int M, int N, int K, size_t ldy, int epilogue) {
    constexpr int SB = RT == 1 && NT == 1 ? 4 : 2;  // steps requested together (registers)
    constexpr int kRows = GATED ? 8 : 16;
    __shared__ float s_red[kGemv4Warps][RT][NT][4][32];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int Kp = (K + 31) & ~31, pitch = Kp >> 1;
    const int steps = (Kp + 127) >> 7;
    const size_t pieces = (size_t)((K + 255) >> 8) * (NV ? 4 : 2);
    const uint8_t *code_ptr[RT][2], *scale_ptr[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const Fp4Operand &w = GATED && h ? w1 : w0;
            const int row = gemv4_row<GATED>((int)blockIdx.x * RT + r, GATED ? g : g + 8 * h);
            const int safe = row < N ? row : N - 1;  // rows past the end are computed from another row and dropped
            code_ptr[r][h] = w.codes + (size_t)safe * pitch + 16 * t;
            scale_ptr[r][h] = w.pieces + scale_piece_offset((size_t)safe, NV ? 4 * (t >> 1) : 0, pieces);
        }

    uint4 code[2][SB][RT][2];
    uint32_t scale[2][SB][RT][2];
    auto request = [&](uint4 (&c)[SB][RT][2], uint32_t (&s)[SB][RT][2], int first) {
#pragma unroll
        for (int b = 0; b < SB; ++b) {
            const int step = first + b * kGemv4Warps;
            const bool in = step < steps, whole = in && step * 64 + 16 * t < pitch;
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    c[b][r][h] = whole ? ld_stream_16(code_ptr[r][h] + (size_t)step * 64) : make_uint4(0, 0, 0, 0);
                    s[b][r][h] = in ? __ldg(reinterpret_cast<const uint32_t *>(scale_ptr[r][h] + (size_t)step * (NV ? 1024 : 512))) : 0u;
                }
        }
    };
    request(code[0], scale[0], warp);
    pdl_wait();  // activations may be the previous kernel's output, which may also still read y

    int n_terms = 1;
    for (int m = lane; m < M; m += 32) n_terms = counts[m];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const int other = __shfl_xor_sync(0xFFFFFFFFu, n_terms, o);
        n_terms = other > n_terms ? other : n_terms;
    }
    int top = 0, windows = 1;
    if constexpr (!NV) {
        top = w0.params->max_byte;
        int low = w0.params->min_byte;
        if constexpr (GATED) {
            top = w1.params->max_byte > top ? w1.params->max_byte : top;
            low = w1.params->min_byte < low ? w1.params->min_byte : low;
        }
        windows = top >= low ? (top - low) / kMxWindow + 1 : 1;
    }

    float total[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[r][n][i] = 0.0f;

    const int passes = n_terms * windows;
    for (int pass = 0; pass < passes; ++pass) {
        const int term = pass / windows, window = pass % windows;
        const int first = top - (kMxWindow - 1) - kMxWindow * window;  // MX: the byte of 2^-14 in this window
        const uint16_t *xrow[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) xrow[n] = 8 * n + g < M ? terms + ((size_t)term * M + 8 * n + g) * Kp + 32 * t : nullptr;
        float acc[RT][NT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;
        auto multiply = [&](uint4 (&c)[SB][RT][2], uint32_t (&s)[SB][RT][2], int first_step) {
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                const int step = first_step + b * kGemv4Warps;
                if (step >= steps) break;
                const int k = step * 128 + 32 * t;
                uint4 xv[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        xv[n][q] = xrow[n] && k < Kp ? __ldg(reinterpret_cast<const uint4 *>(xrow[n] + step * 128) + q) : make_uint4(0, 0, 0, 0);
                uint32_t f[RT][2][2];
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (NV) {  // blocks 2t and 2t + 1 of the step's 8: half t % 2 of word t / 2, which this lane loaded
                            const uint32_t two = cvt_f16x2_e4m3(s[b][r][h] >> (16 * (t & 1)));
                            f[r][h][0] = dup_lo(two);
                            f[r][h][1] = dup_hi(two);
                        } else {
                            f[r][h][0] = f[r][h][1] = mx_scale_f16x2(s[b][r][h], t, first);
                        }
                    }
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // words of 8 codes
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint4 &ca = c[b][r][0], &cb = c[b][r][1];
                        const uint32_t wa = q == 0 ? ca.x : q == 1 ? ca.y : q == 2 ? ca.z : ca.w, wb = q == 0 ? cb.x : q == 1 ? cb.y : q == 2 ? cb.z : cb.w;
                        uint32_t ha[4], hb[4];
                        cvt_f16x8_e2m1(wa, ha);
                        cvt_f16x8_e2m1(wb, hb);
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            ha[p] = mul_f16x2(ha[p], f[r][0][q >> 1]);
                            hb[p] = mul_f16x2(hb[p], f[r][1][q >> 1]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_f16_16816(acc[r][n], ha[0], hb[0], ha[1], hb[1], xv[n][q].x, xv[n][q].y);
                            mma_f16_16816(acc[r][n], ha[2], hb[2], ha[3], hb[3], xv[n][q].z, xv[n][q].w);
                        }
                    }
                }
            }
        };
        for (int step = warp; step < steps; step += 2 * SB * kGemv4Warps) {
            const int second = step + SB * kGemv4Warps;
            request(code[1], scale[1], second);
            multiply(code[0], scale[0], step);
            // (behind the last steps: the first ones again, for a pass that may follow)
            const int third = second + SB * kGemv4Warps;
            if (third < steps || pass + 1 < passes) request(code[0], scale[0], third < steps ? third : warp);
            multiply(code[1], scale[1], second);
        }
        // weight of this pass's sums: 2^-11 or 2^-32 for each term, 2^-28 for each window
        const float weight = pass == 0 ? 1.0f : ldexpf(1.0f, -(n_terms == 3 ? 11 : 32) * term - kMxWindow * window);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[r][n][i] = __fmaf_rn(acc[r][n][i], weight, total[r][n][i]);
    }

#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_red[warp][r][n][i][lane] = total[r][n][i];
    __syncthreads();

    // accumulator (lane, i) of token group n: row (lane / 4) + (i >= 2 ? 8 : 0), token 8 n + 2 (lane % 4) + (i & 1)
    const float a0 = NV ? w0.params->tensor_scale : 1.0f, a1 = GATED && NV ? w1.params->tensor_scale : 1.0f;
    for (int o = threadIdx.x; o < kRows * RT * 8 * NT; o += kGemv4Warps * 32) {
        const int i = o % kRows, r = o / kRows % RT, m = o / (kRows * RT);
        const int n = gemv4_row<GATED>((int)blockIdx.x * RT + r, i);
        if (n >= N || m >= M) continue;
        const int ln = (i & 7) * 4 + ((m & 7) >> 1), lo = (m & 1) + ((i & 8) ? 2 : 0);
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int w = 0; w < kGemv4Warps; ++w) {
            s0 += s_red[w][r][m >> 3][lo][ln];
            if constexpr (GATED) s1 += s_red[w][r][m >> 3][2 + (m & 1)][ln];
        }
        // back from the token's power of two and, for MX, from the window's: the first window has its largest scale, 2^(top - 127), at 2^13
        const int back = exps[m] + (NV ? 0 : top - 127 - 13);
        float v = ldexpf(s0, back) * a0;
        if (w0.bias) v += w0.bias[n];
        if constexpr (GATED) {
            float u = ldexpf(s1, back) * a1;
            if (w1.bias) u += w1.bias[n];
            v = v / (1.0f + __expf(-v)) * u;
        } else if (epilogue == SHREWQ_EPILOGUE_RELU) {
            v = fmaxf(v, 0.0f);
        }
        store_out<YT>(y + (size_t)m * ldy + n, v);
    }
}

// ---- a handle's copy of the scales --------------------------------------------------------------------------------------------------
// scales [N][blocks] -> pieces (128 rows x 4 blocks, 512 bytes, out to whole 256 columns and 128 rows; scale 1 in the padding), the
// tensor scale, and for MX the range of the bytes (NaN apart; params starts with max_byte 0 and min_byte -1).  alpha[n]: what a sum of
// channel n is multiplied by, the tensor scales of both operands.
template <bool NV>
__global__ void __launch_bounds__(256)
fp4_scale_pieces_kernel(const uint8_t *__restrict__ scales, const float *g, size_t N, size_t blocks, size_t pieces, uint8_t *__restrict__ out,
                        Fp4Params *params, float x_scale, float *__restrict__ alpha) {
    const size_t total = (N + 127) / 128 * 128 * pieces;  // words
    int top = 0, low = 255;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t row = i / pieces, piece = i % pieces;
        uint32_t word = 0;
        for (int j = 0; j < 4; ++j) {
            const size_t b = piece * 4 + j;
            uint32_t byte = NV ? kE4m3One : kE8m0One;
            if (row < N && b < blocks) {
                byte = scales[row * blocks + b];
                if (byte != 255u) {
                    top = (int)byte > top ? (int)byte : top;
                    low = (int)byte < low ? (int)byte : low;
                }
            }
            word |= byte << (8 * j);
        }
        *reinterpret_cast<uint32_t *>(out + scale_piece_offset(row, piece * 4, pieces)) = word;
    }
    if constexpr (!NV) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const int a = __shfl_xor_sync(0xFFFFFFFFu, top, o), b = __shfl_xor_sync(0xFFFFFFFFu, low, o);
            top = a > top ? a : top;
            low = b < low ? b : low;
        }
        if ((threadIdx.x & 31) == 0) {
            atomicMax(reinterpret_cast<unsigned int *>(&params->max_byte), (unsigned int)top);
            atomicMin(reinterpret_cast<unsigned int *>(&params->min_byte), (unsigned int)low);
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        params->tensor_scale = NV ? *g : 1.0f;
        params->x_scale = x_scale;
    }
    for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < N; n += (size_t)gridDim.x * 256) alpha[n] = NV ? *g * x_scale : 1.0f;
}

}  // namespace
}  // namespace shrewq
