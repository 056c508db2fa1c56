// Forward of a layer with 4-bit microscaled weights for up to 4 tokens, sm_100a: warp-level MMA on f16 operands.
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
// Activations are f16 too: staging scales every token by a power of two to [2^14, 2^15) and forms f16 terms: bf16 values down to 2^-32
// of their token's largest are exact in the first; where a token has smaller ones a second term holds what the first left, times 2^32.
// f32 values take three terms of 11 bits each.  The kernel passes over the codes once for every term that any token needs, and adds the
// passes' sums with their weights in f32.  Products are exact, sums are f32.
//
// Mapping.  One CTA of 16 warps an SM walks over tiles of 16 rows (GATED: 8 gate rows and the 8 up rows of the same channels); the
// warps deal the k range in steps of 128 codes.  mma.sync.m16n8k16 with the weights as the A operand: lane (g = lane / 4, t = lane % 4)
// takes 16 bytes = 32 consecutive codes (one MX block, two NV blocks: the scale is the lane's own) of rows g and g + 8 and the 32
// activations of the same k for token g; MMA step i uses the codes 4i .. 4i+3 of that run for A and B alike.
// Codes and scales come by cp.async, every lane its own bytes into its own slots of a ring, several steps ahead and across tiles: no
// register holds a byte in flight, no barrier guards one, and an SM has some 60 KB on their way.  The rows of a tile are 4 neighbours
// each from the 4 groups of 32 that share 16 bytes of scales in the handle's copy (scale_piece_offset): scale sectors are used whole.
// Activations: every CTA stages them in its shared memory while its first codes are on their way: one launch, no workspace.  (From 5 tokens
// on the tcgen05 kernels: an m16n8k16 of mma.sync holds its tensor pipe for 32 cycles, which one group of 8 tokens just allows.)
// The warps' sums of a tile meet in shared memory in a fixed order.
//
// Programmatic dependent launch: the ring is filled before the wait for the previous kernel.
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

constexpr int kGemv4Warps = 16, kGemv4Threads = kGemv4Warps * 32;
constexpr int kGemv4Depth = 4;         // steps of the ring
constexpr int kGemv4SlotBytes = 40;    // of a lane and step: 16 bytes of codes of two rows, a scale word for each
constexpr int kGemv4RingBytes = kGemv4Warps * kGemv4Depth * 32 * kGemv4SlotBytes;
constexpr int kGemv4MaxStaged = 4;     // tokens that a CTA stages ...
constexpr int kGemv4StagedBytes = 96 * 1024;  // ... in at most this much shared memory
constexpr int kMxWindow = 28;          // octaves of MX scales that one pass takes

// What the kernels need of one weight matrix (device pointers; params and pieces belong to the handle)
struct Fp4Operand {
    const uint8_t *codes;    // [N][pitch]
    const uint8_t *pieces;   // scales in the order of scale_piece_offset
    const Fp4Params *params;
    const float *bias;
};

// ---- activations -> f16 terms -----------------------------------------------------------------------------------------------
// Terms of f32 and bf16 activations, and the power of two between them
template <typename T>
struct XTerms {
    static constexpr int kMost = sizeof(T) == 4 ? 3 : 2;
    static constexpr int kOctaves = sizeof(T) == 4 ? 11 : 32;
};
template <typename T>
__device__ __forceinline__ void load_token8(const T *row, int i, int K, int vec_ok, float *v) {
    if (vec_ok && i * 8 + 8 <= K) load_vec8<T>(row + i * 8, v);
    else load_guarded8<T>(row + i * 8, i * 8 < K ? (size_t)(K - i * 8) : 0, v);
}
// largest exponent field of finite values among v[8] and top
__device__ __forceinline__ unsigned int top_exponent(const float *v, unsigned int top) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned int e = (__float_as_uint(v[j]) >> 23) & 0xFFu;
        top = e < 255u && e > top ? e : top;
    }
    return top;
}
__device__ __forceinline__ unsigned int warp_max(unsigned int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned int other = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = other > v ? other : v;
    }
    return v;
}
// v[8] -> terms of 8 f16; returns whether the first term left anything.  Infinities and NaNs stay what they are in the first term and
// are 0 in the others.  top: the token's largest exponent field: x is multiplied by 2^(141 - top), as two factors that are ordinary numbers
template <typename T>
__device__ __forceinline__ bool f16_terms(float *v, unsigned int top, uint4 *out) {
    const int up = 141 - (int)top;  // -113 .. 141
    const float f0 = __uint_as_float((uint32_t)(127 + (up > 100 ? 100 : up)) << 23), f1 = __uint_as_float((uint32_t)(127 + (up > 100 ? up - 100 : 0)) << 23);
    const float next = sizeof(T) == 4 ? 2048.0f : 4294967296.0f;
    bool more = false;
    uint32_t w[XTerms<T>::kMost][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = v[2 * j] * f0 * f1, b = v[2 * j + 1] * f0 * f1;
#pragma unroll
        for (int t = 0; t < XTerms<T>::kMost; ++t) {
            w[t][j] = pack_f16x2_rn(b, a);
            float ha, hb;
            f32x2_of_f16x2(w[t][j], ha, hb);
            a = ha - ha == 0.0f ? (a - ha) * next : 0.0f;
            b = hb - hb == 0.0f ? (b - hb) * next : 0.0f;
            if (t == 0) more = more || a != 0.0f || b != 0.0f;
        }
    }
#pragma unroll
    for (int t = 0; t < XTerms<T>::kMost; ++t) out[t] = make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
    return more;
}

// For gemm_fp4_f16_kernels.cuh: a CTA a token.  terms: [kMost][M][Kp] f16 (Kp = K to whole 32s, zeros beyond K); exps[m]: the power of two that
// the token was divided by; counts[m]: terms in use.
template <typename T>
__global__ void __launch_bounds__(256)
stage_f16_kernel(const T *x, int M, int K, int Kp, int vec_ok, uint4 *__restrict__ terms, int *__restrict__ exps, int *__restrict__ counts) {
    pdl_launch_dependents();
    __shared__ unsigned int s_max[8], s_more[8];
    const int m = blockIdx.x, threads = (int)blockDim.x, warps = threads >> 5, groups = Kp >> 3;
    const size_t plane = (size_t)M * groups;
    pdl_wait();
    const T *row = x + (size_t)m * K;
    unsigned int top = 0, more = 0;
    for (int i = threadIdx.x; i < groups; i += threads) {
        float v[8];
        load_token8<T>(row, i, K, vec_ok, v);
        top = top_exponent(v, top);
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = s_max[w] > top ? s_max[w] : top;
    for (int i = threadIdx.x; i < groups; i += threads) {
        float v[8];
        load_token8<T>(row, i, K, vec_ok, v);
        uint4 out[XTerms<T>::kMost];
        more |= f16_terms<T>(v, top, out) ? 1u : 0u;
#pragma unroll
        for (int t = 0; t < XTerms<T>::kMost; ++t) terms[t * plane + (size_t)m * groups + i] = out[t];
    }
    more = warp_max(more);
    if ((threadIdx.x & 31) == 0) s_more[threadIdx.x >> 5] = more;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 0; w < warps; ++w) more |= s_more[w];
        exps[m] = (int)top - 141;
        counts[m] = more ? XTerms<T>::kMost : 1;
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

// M <= kGemv4MaxStaged
template <bool NV, bool GATED, typename T, typename YT>
__global__ void __launch_bounds__(kGemv4Threads, 1)
gemv_fp4_kernel(Fp4Operand w0, Fp4Operand w1, const T *x, int vec_ok, YT *__restrict__ y, int M, int N, int K, size_t ldy, int epilogue) {
    constexpr int kRows = GATED ? 8 : 16;
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem);  // ring, then the staged activations
    __shared__ float s_red[2][kGemv4Warps][4][32];
    __shared__ unsigned int s_max[kGemv4MaxStaged][kGemv4Warps], s_more[kGemv4Warps];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int Kp = (K + 31) & ~31, pitch = Kp >> 1;
    const int steps = (Kp + 127) >> 7;
    const size_t pieces = (size_t)((K + 255) >> 8) * (NV ? 4 : 2);
    const int tiles = ((N + 127) >> 7) * (GATED ? 16 : 8);
    const int mine = (steps - warp + kGemv4Warps - 1) / kGemv4Warps;  // this warp's steps of a tile (not negative: warp < 16)

    // ---- the ring: item i of this warp is its step i % mine of the CTA's tile i / mine ----
    const uint32_t ring = smem_offset(smem) + (uint32_t)((warp * kGemv4Depth * 32 + lane) * 16);
    constexpr uint32_t kRowH = kGemv4Warps * kGemv4Depth * 32 * 16;   // codes of rows g, codes of rows g + 8, scale words of both
    const uint32_t ring_scales = smem_offset(smem) + 2 * kRowH + (uint32_t)((warp * kGemv4Depth * 32 + lane) * 8);
    const uint8_t *code_ptr[2], *scale_ptr[2];
    int next_tile = (int)blockIdx.x, next_step = warp, slot_in = 0;
    auto aim = [&](int tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const Fp4Operand &w = GATED && h ? w1 : w0;
            const int row = gemv4_row<GATED>(tile, GATED ? g : g + 8 * h);
            const int safe = row < N ? row : N - 1;  // rows past the end are computed from another row and dropped
            code_ptr[h] = w.codes + (size_t)safe * pitch + 16 * t;
            scale_ptr[h] = w.pieces + scale_piece_offset((size_t)safe, NV ? 4 * (t >> 1) : 0, pieces);
        }
    };
    // requests the next item, or nothing behind the last one; every call closes a group of copies
    auto request = [&]() {
        if (next_step < steps && next_tile < tiles) {
            const bool in = next_step * 64 + 16 * t < pitch;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                copy_async_16(ring + h * kRowH + slot_in * 512, code_ptr[h] + (in ? (size_t)next_step * 64 : 0), in);
                copy_async_4(ring_scales + slot_in * 256 + h * 4, scale_ptr[h] + (size_t)next_step * (NV ? 1024 : 512), true);
            }
            slot_in = slot_in + 1 == kGemv4Depth ? 0 : slot_in + 1;
            next_step += kGemv4Warps;
            if (next_step >= steps) {
                next_step = warp;
                next_tile += (int)gridDim.x;
                if (next_tile < tiles) aim(next_tile);
            }
        }
        copy_async_commit();
    };
    // passes over a tile's codes: a ring that is read more than once would have to be filled again, so the passes are outermost
    aim(next_tile);
#pragma unroll
    for (int i = 0; i < kGemv4Depth - 1; ++i) request();
    pdl_wait();  // activations may be the previous kernel's output, which may also still read y

    // ---- activations ----
    int n_terms = 1;
    const uint4 *sx = reinterpret_cast<const uint4 *>(smem + kGemv4RingBytes);  // [terms][steps][4][4 t][M]
    unsigned int tops[kGemv4MaxStaged];
    {
        const int groups = steps << 4;
#pragma unroll
        for (int m = 0; m < kGemv4MaxStaged; ++m) {
            tops[m] = 0;
            if (m < M)
                for (int i = threadIdx.x; i < groups; i += kGemv4Threads) {
                    float v[8];
                    load_token8<T>(x + (size_t)m * K, i, K, vec_ok, v);
                    tops[m] = top_exponent(v, tops[m]);
                }
            tops[m] = warp_max(tops[m]);
            if (lane == 0) s_max[m][warp] = tops[m];
        }
        __syncthreads();
        unsigned int more = 0;
        uint4 *dst = reinterpret_cast<uint4 *>(smem + kGemv4RingBytes);
#pragma unroll
        for (int m = 0; m < kGemv4MaxStaged; ++m) {
            for (int w = 0; w < kGemv4Warps; ++w) tops[m] = s_max[m][w] > tops[m] ? s_max[m][w] : tops[m];
            if (m < M)
                for (int i = threadIdx.x; i < groups; i += kGemv4Threads) {
                    float v[8];
                    load_token8<T>(x + (size_t)m * K, i, K, vec_ok, v);
                    uint4 out[XTerms<T>::kMost];
                    more |= f16_terms<T>(v, tops[m], out) ? 1u : 0u;
#pragma unroll
                    for (int e = 0; e < XTerms<T>::kMost; ++e)
                        dst[(size_t)(((e * steps + (i >> 4)) * 4 + (i & 3)) * 4 + ((i >> 2) & 3)) * M + m] = out[e];
                }
        }
        more = warp_max(more);
        if (lane == 0) s_more[warp] = more;
        __syncthreads();
        for (int w = 0; w < kGemv4Warps; ++w) n_terms = s_more[w] ? XTerms<T>::kMost : n_terms;
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
    const int passes = n_terms * windows;

    // One step: codes (two rows), scale words, activations -> acc
    auto multiply = [&](float (&acc)[4], uint4 ca, uint4 cb, uint32_t sa, uint32_t sb, int step, int term, int first) {
        uint4 xv[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) xv[q] = g < M ? sx[(size_t)(((term * steps + step) * 4 + q) * 4 + t) * M + g] : make_uint4(0, 0, 0, 0);
        uint32_t f[2][2];
        if constexpr (NV) {  // blocks 2t and 2t + 1 of the step's 8: half t % 2 of word t / 2, which this lane loaded
            const uint32_t a2 = cvt_f16x2_e4m3(sa >> (16 * (t & 1))), b2 = cvt_f16x2_e4m3(sb >> (16 * (t & 1)));
            f[0][0] = dup_lo(a2);
            f[0][1] = dup_hi(a2);
            f[1][0] = dup_lo(b2);
            f[1][1] = dup_hi(b2);
        } else {
            f[0][0] = f[0][1] = mx_scale_f16x2(sa, t, first);
            f[1][0] = f[1][1] = mx_scale_f16x2(sb, t, first);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // words of 8 codes
            uint32_t ha[4], hb[4];
            cvt_f16x8_e2m1(q == 0 ? ca.x : q == 1 ? ca.y : q == 2 ? ca.z : ca.w, ha);
            cvt_f16x8_e2m1(q == 0 ? cb.x : q == 1 ? cb.y : q == 2 ? cb.z : cb.w, hb);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                ha[p] = mul_f16x2(ha[p], f[0][q >> 1]);
                hb[p] = mul_f16x2(hb[p], f[1][q >> 1]);
            }
            mma_f16_16816(acc, ha[0], hb[0], ha[1], hb[1], xv[q].x, xv[q].y);
            mma_f16_16816(acc, ha[2], hb[2], ha[3], hb[3], xv[q].z, xv[q].w);
        }
    };

    const float alpha0 = NV ? w0.params->tensor_scale : 1.0f, alpha1 = GATED && NV ? w1.params->tensor_scale : 1.0f;
    int slot = 0, turn = 0;
    for (int tile = (int)blockIdx.x; tile < tiles; tile += (int)gridDim.x, turn ^= 1) {
        float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < mine; ++s) {
            request();
            copy_async_wait<kGemv4Depth - 1>();
            const uint8_t *at = smem + (size_t)(warp * kGemv4Depth * 32 + slot * 32 + lane) * 16;
            const uint4 ca = *reinterpret_cast<const uint4 *>(at), cb = *reinterpret_cast<const uint4 *>(at + kRowH);
            const uint2 sc = *reinterpret_cast<const uint2 *>(smem + 2 * kRowH + (size_t)(warp * kGemv4Depth * 32 + slot * 32 + lane) * 8);
            slot = slot + 1 == kGemv4Depth ? 0 : slot + 1;
            const int step = warp + s * kGemv4Warps;
            if (passes == 1) {
                multiply(total, ca, cb, sc.x, sc.y, step, 0, top - (kMxWindow - 1));
            } else {
                for (int pass = 0; pass < passes; ++pass) {
                    const int term = pass / windows, window = pass % windows;
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    multiply(acc, ca, cb, sc.x, sc.y, step, term, top - (kMxWindow - 1) - kMxWindow * window);
                    // weight of this pass's sums: 2^-11 or 2^-32 for each term, 2^-28 for each window
                    const float weight = ldexpf(1.0f, -XTerms<T>::kOctaves * term - kMxWindow * window);
#pragma unroll
                    for (int i = 0; i < 4; ++i) total[i] = __fmaf_rn(acc[i], weight, total[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s_red[turn][warp][i][lane] = total[i];
        __syncthreads();  // (with two buffers a warp writes this one again only behind the next barrier)

        // accumulator (lane, i): row (lane / 4) + (i >= 2 ? 8 : 0), token 2 (lane % 4) + (i & 1)
        for (int o = threadIdx.x; o < kRows * M; o += kGemv4Threads) {
            const int i = o % kRows, m = o / kRows;
            const int n = gemv4_row<GATED>(tile, i);
            if (n >= N) continue;
            const int ln = (i & 7) * 4 + (m >> 1), lo = (m & 1) + ((i & 8) ? 2 : 0);
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int w = 0; w < kGemv4Warps; ++w) {
                s0 += s_red[turn][w][lo][ln];
                if constexpr (GATED) s1 += s_red[turn][w][2 + (m & 1)][ln];
            }
            const int exponent = (int)(m == 0 ? tops[0] : m == 1 ? tops[1] : m == 2 ? tops[2] : tops[3]) - 141;
            // back from the token's power of two and, for MX, from the window's: the first window has its largest scale, 2^(top - 127), at 2^13
            const int back = exponent + (NV ? 0 : top - 127 - 13);
            float v = ldexpf(s0, back) * alpha0;
            if (w0.bias) v += w0.bias[n];
            if constexpr (GATED) {
                float u = ldexpf(s1, back) * alpha1;
                if (w1.bias) u += w1.bias[n];
                v = v / (1.0f + __expf(-v)) * u;
            } else if (epilogue == SHREWQ_EPILOGUE_RELU) {
                v = relu_nan(v);
            }
            store_out<YT>(y + (size_t)m * ldy + n, v);
        }
    }
    copy_async_wait<0>();
}

// ---- a handle's copy of the scales --------------------------------------------------------------------------------------------------
// scales [N][blocks] -> pieces (128 rows x 4 blocks, 512 bytes, out to whole 256 columns and 128 rows; scale 1 in the padding), the
// tensor scale, and for MX the range of the bytes (NaN apart; params starts with max_byte 0 and min_byte -1).  alpha[n]: what a sum of
// channel n is multiplied by, the tensor scales of both operands.
template <bool NV>
__global__ void __launch_bounds__(256)
fp4_scale_pieces_kernel(const uint8_t *scales, const float *g, size_t N, size_t blocks, size_t pieces, uint8_t *__restrict__ out,
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
