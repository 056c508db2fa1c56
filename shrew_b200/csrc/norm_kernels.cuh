// What stands between two blocks of a residual network, in one pass over the rows:
//
//   b = branch                          the output of the block before             (no branch: b is left out)
//   b = norm_post(b)                    the norm after that block                   (optional)
//   b = gate * b                        one value a channel, a token or an element  (optional)
//   r = residual_scale * x + branch_scale * b       the residual stream
//   h = norm_pre(r)                     the norm before the next block              (optional)
//
//   RMS:   norm(v) = v / sqrt(mean(v^2) + eps) * weight (+ bias)
//   layer: norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) * weight (+ bias)
//
// Everything is computed in f32; r is rounded once to the type of x, and h is formed from the r before that rounding (nearer to the
// formula than a norm that reads the stored r back), rounded once to its own type.  The variance of a layer norm is summed from the
// centred values, which stay in registers: no cancellation for rows far from zero.
//
// Memory-bound: x and branch are read once and r and h written once.  A row lives in the registers of a warp (up to 1024 columns) or of a
// CTA (V groups of 8 columns a thread), so the two statistics cost no second read; above 16384 columns (V = 4 with 64 registers a thread) 320 to 612
// bytes a thread are spilled.  The weights come through L1, which the rows' streaming loads leave to them.
// Measured (f32 stream, bf16 branch and gate of channels, norms before and after, bf16 out): 4096 rows of 4096 45 us, 4.5 TB/s of half reads and half
// writes; 2048 rows of 16384 106 us, 3.8 TB/s; 1024 rows of 32768 127 us, 3.2 TB/s.  A row is two sums of a CTA, one after the other, with four
// rows of 4096 an SM under way and no load of the next rows meanwhile (registers are taken; shared memory is not used for it).
//
// Device code only (no launch syntax; PTX behind ptx_fp4.cuh and ptx_small.cuh): also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "fp4_kernels.cuh"

namespace shrewq {
namespace {

enum NormKindDev { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum GateKind { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct NormArgs {
    const void *x, *branch, *gate;       // branch null: none
    size_t ldx, ldb, ldg;                // row strides, elements
    const float *post_w, *post_b, *pre_w, *pre_b;  // null: 1 and 0
    void *r, *h;                         // [M][D], null: not wanted
    size_t M;
    int D;
    int post, pre, gate_kind;
    float post_eps, pre_eps, residual_scale, branch_scale;
    int vec;                             // every row of every operand starts on the boundary of a whole group and D is a multiple of 8
};

// eight f32 parameters from column c on (cached in L1)
__device__ __forceinline__ void load_params8(const float *p, int c, int D, int vec, float otherwise, float *v) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = otherwise;
    } else if (vec) {
        const float4 a = *reinterpret_cast<const float4 *>(p + c), b = *(reinterpret_cast<const float4 *>(p + c) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < D ? p[c + i] : 0.0f;
    }
}

// sum over the threads of a row: a warp, or the whole CTA through s_red (two buffers taken in turn, one barrier a sum)
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float (*s_red)[32], int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if constexpr (!WARP) {
        const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) s_red[turn][threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? s_red[turn][lane] : 0.0f;
        turn ^= 1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    }
    return v;
}

// v[V][8] (columns 8 (u * T + t) .. + 7, zero beyond D) -> normalised in place
template <int V, bool WARP>
__device__ __forceinline__ void norm_row(float (*v)[8], int t, int T, int D, int kind, float eps, const float *w, const float *b, int vec,
                                         float (*s_red)[32], int &turn) {
    const float inv_d = __fdiv_rn(1.0f, (float)D);
    if (kind == kNormLayer) {
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < V; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[u][i];
        const float mean = row_sum<WARP>(s, s_red, turn) * inv_d;
#pragma unroll
        for (int u = 0; u < V; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = (u * T + t) * 8 + i < D ? v[u][i] - mean : 0.0f;
    }
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __fmaf_rn(v[u][i], v[u][i], s);
    const float inv = rsqrtf(row_sum<WARP>(s, s_red, turn) * inv_d + eps);
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int c = (u * T + t) * 8;
        if (c >= D) continue;
        float wv[8], bv[8];
        load_params8(w, c, D, vec, 1.0f, wv);
        load_params8(b, c, D, vec, 0.0f, bv);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = __fmaf_rn(v[u][i] * inv, wv[i], bv[i]);
    }
}

template <typename T>
__device__ __forceinline__ void load_row8(const T *row, int c, int D, int vec, float *v) {
    if (c >= D) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if (vec) load_vec8<T>(row + c, v);
    else load_guarded8<T>(row + c, (size_t)(D - c), v);
}
// eight values that every row uses again: through L1, which the rows' own loads pass by (a gate of channels from L2 for every row:
// 4096 rows of 4096 in 47.7 us instead of 44.3)
__device__ __forceinline__ void load_shared8(const float *p, float *v) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load_shared8(const __nv_bfloat16 *p, float *v) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
}

template <typename T>
__device__ __forceinline__ void store_row8(T *row, int c, int D, int vec, const float *v) {
    if (c >= D) return;
    if (vec) store_vec8<T>(row + c, v);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < D) from_f32(v[i], row + c + i);
}

// WARP: a warp a row (blockDim.x / 32 rows a CTA); else a CTA a row.
template <typename TX, typename TB, typename TY, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
residual_norm_kernel(NormArgs a) {
    pdl_launch_dependents();
    __shared__ float s_red[2][32];
    int turn = 0;
    const int T = WARP ? 32 : (int)blockDim.x, t = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
    const size_t per_cta = WARP ? blockDim.x >> 5 : 1;
    pdl_wait();
    for (size_t m = (size_t)blockIdx.x * per_cta + (WARP ? threadIdx.x >> 5 : 0); m < a.M; m += (size_t)gridDim.x * per_cta) {
        float r[V][8];
        const TX *x = static_cast<const TX *>(a.x) + m * a.ldx;
#pragma unroll
        for (int u = 0; u < V; ++u) load_row8<TX>(x, (u * T + t) * 8, a.D, a.vec, r[u]);
        if (a.branch) {
            float b[V][8];
            const TB *br = static_cast<const TB *>(a.branch) + m * a.ldb;
#pragma unroll
            for (int u = 0; u < V; ++u) load_row8<TB>(br, (u * T + t) * 8, a.D, a.vec, b[u]);
            if (a.post != kNormNone) norm_row<V, WARP>(b, t, T, a.D, a.post, a.post_eps, a.post_w, a.post_b, a.vec, s_red, turn);
            const TB *gate = static_cast<const TB *>(a.gate);
            const float token = a.gate_kind == kGateToken ? to_f32(gate[m * a.ldg]) : 1.0f;
#pragma unroll
            for (int u = 0; u < V; ++u) {
                float g[8];
                const int c = (u * T + t) * 8;
                if (a.gate_kind == kGateChannel && a.vec && c < a.D) load_shared8(gate + c, g);
                else if (a.gate_kind == kGateChannel) load_row8<TB>(gate, c, a.D, a.vec, g);
                else if (a.gate_kind == kGateFull) load_row8<TB>(gate + m * a.ldg, c, a.D, a.vec, g);
                else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] = token;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) r[u][i] = __fmaf_rn(a.branch_scale, b[u][i] * g[i], a.residual_scale * r[u][i]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < V; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) r[u][i] *= a.residual_scale;
        }
        if (a.r) {
#pragma unroll
            for (int u = 0; u < V; ++u) store_row8<TX>(static_cast<TX *>(a.r) + m * (size_t)a.D, (u * T + t) * 8, a.D, a.vec, r[u]);
        }
        if (a.h) {
            norm_row<V, WARP>(r, t, T, a.D, a.pre, a.pre_eps, a.pre_w, a.pre_b, a.vec, s_red, turn);
#pragma unroll
            for (int u = 0; u < V; ++u) store_row8<TY>(static_cast<TY *>(a.h) + m * (size_t)a.D, (u * T + t) * 8, a.D, a.vec, r[u]);
        }
    }
}

}  // namespace
}  // namespace shrewq
