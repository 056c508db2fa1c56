// Forward of a layer with 4-bit microscaled weights and activations as they come, on the tensor cores (tcgen05.mma kind::f16 in bf16),
// sm_100a only.
//
//   y[m,n] = epi( alpha[n] * sum_k (w code * w scale)[n,k] x[m,k] + bias[n] )
//
// code * scale is exact in bf16: an E2M1 code has two significant bits, an E8M0 scale is a power of two of bf16's own exponent range, an E4M3
// scale has four bits.  bf16 activations are used as they are; f32 ones come as three bf16 terms (8 + 8 + 8 bits, truncated one after
// the other: exact), three MMAs a step (XT = 3).  Their sums keep four accumulators: the leading terms' go to three in turn, stage by stage, and those
// of the two others, 2^-8 and less of them, to one of their own, where they do not drown in the sum of the leading ones; all are added in f32 at the
// end.  (In one accumulator, which loses what is below its last place at every step, k = 11008 was 2.7e-5 off.)  bf16 activations have two accumulators in
// turn in tiles of 64 tokens (sums of 11008 NV products 4.3e-6 -> 1.8e-6 off, and 4096 x 11008 16.1 -> 14.9 us; three: 1.0e-6, 15.4 us) and one in larger
// ones, where a second costs a stage of the ring (128 tokens of gated 11008 x 4096: 34.9 -> 40.4 us).
//
// Mapping.  D[128 x TOK] += A[128 x 16] * B[TOK x 16]^T: A = 128 weight rows, widened by converter warps and written to TENSOR MEMORY with
// tcgen05.st; B = a tile of tokens in shared memory (TMA, 128-byte swizzle); D = f32 accumulators in tensor memory (lane = channel).
// A stage holds 128 codes of k a row (64 bytes, TMA with the 64-byte swizzle) and the scale pieces of its rows.  Widening: one
// conversion makes two codes f16, two more f32, a pack makes them bf16 and one packed multiplication applies the scale: 2.5 issue
// slots a code, of which one on the 16-lane ALU pipe (moving the bits from f16 to bf16 by shift and masks takes two there).
// GATED: 64 gate rows and 64 up rows of the same channels, interleaved lane by lane in tensor memory.
// The k range of a tile may be split over a cluster (tcgen05_cluster_epilogue.cuh).
//
// Warp roles: warp 0 = TMA producer, warp 1 = tensor-memory allocation and MMA issue, then 3 groups of 4 converter warps (a group owns the
// stages s with s % 3 == its number), which run the epilogue too.  full[s] -> converters -> aready[s] -> MMA -> empty[s]; bounded waits.
// Programmatic dependent launch: weights and scales of the first stages are requested before the wait for the previous kernel.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "../../include/shrewq.h"
#include "fp4_kernels.cuh"
#include "ptx_small.cuh"
#include "ptx_tcgen05.cuh"
#include "tcgen05_cluster_epilogue.cuh"
#include "tcgen05_common.cuh"

namespace shrewq {
namespace {

constexpr int kW4Groups = 3;
constexpr int kW4Threads = 64 + 128 * kW4Groups;
constexpr uint32_t kTimeoutW4 = 6;  // DeviceStatus::timeout_flag of this kernel

constexpr int kW4StageK = 128;  // codes of k a stage
template <int TOK, int XT, bool NV, bool GATED>
struct W4Cfg {
    static constexpr int kCodeRow = kW4StageK / 2;                               // bytes of codes of a row in a stage
    static constexpr int kCodeBytes = 128 * kCodeRow;
    static constexpr int kPieces = NV ? 2 : 1;      // scale pieces of a row group a stage
    static constexpr int kMats = GATED ? 2 : 1;
    static constexpr int kScaleBytes = kMats * kPieces * 512;
    static constexpr int kXBox = TOK * 128;                               // 64 bf16 of every token
    static constexpr int kXBytes = XT * (kW4StageK / 64) * kXBox;
    static constexpr int kXOff = kCodeBytes;
    static constexpr int kScaleOff = kXOff + kXBytes;
    static constexpr int kStageBytes = (kScaleOff + kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kTxBytes = kCodeBytes + kXBytes + kScaleBytes;
    static constexpr int kACols = kW4StageK / 2;
    static constexpr int kLow = XT == 3 ? 1 : 0, kLeading = XT == 3 ? 3 : TOK == 64 ? 2 : 1, kAccs = kLow + kLeading;  // accumulators: of the low terms, then of the leading ones
    static constexpr int kABase = (kAccs * TOK + 31) / 32 * 32;
    static constexpr int kMaxSmem = (224 * 1024) / kStageBytes, kMaxTmem = (512 - kABase) / kACols;
    static constexpr int kStagesRaw = kMaxSmem < kMaxTmem ? kMaxSmem : kMaxTmem;
    static constexpr int kStages = kStagesRaw > 12 ? 12 : kStagesRaw;
    static constexpr int kSmemBytes = kStages * kStageBytes + 2048;
    static constexpr int kSmemRequest = kSmemBytes > 120 * 1024 ? kSmemBytes : 120 * 1024;  // one CTA an SM: it takes all of tensor memory
    static constexpr int kSlotOff = kW4Groups * kEpiStageBytes;           // received sums behind the staging tiles
    static_assert(kStages >= 3 && kSmemRequest <= 227 * 1024, "stages");
    static_assert(kStages * kStageBytes >= kSlotOff + ClusterEpi<TOK, kEpiPlain>::kSlotBytes, "the epilogue reuses the stages");
};

// 32 codes (16 bytes) and their scale (NV: two) -> 16 packed bf16x2, natural order
__device__ __forceinline__ void widen32(const uint4 c, uint32_t s_lo, uint32_t s_hi, uint32_t *out) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t h[4];
        cvt_f16x8_e2m1(w[q], h);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            float lo, hi;
            f32x2_of_f16x2(h[p], lo, hi);
            out[4 * q + p] = mul_bf16x2(pack_bf16x2_rn(hi, lo), q < 2 ? s_lo : s_hi);
        }
    }
}
// an E8M0 byte as a bf16x2 pair of its value
__device__ __forceinline__ uint32_t e8m0_bf16x2(uint32_t b) {
    const uint32_t h = b == 0 ? 0x0040u : b == 255u ? 0x7FFFu : b << 7;
    return h * 0x10001u;
}
// two E4M3 bytes (low half of a word) as two bf16x2 pairs
__device__ __forceinline__ void e4m3_bf16x2(uint32_t two, uint32_t &first, uint32_t &second) {
    float a, b;
    f32x2_of_f16x2(cvt_f16x2_e4m3(two), a, b);
    first = pack_bf16x2_rn(a, a);
    second = pack_bf16x2_rn(b, b);
}

// f32 or bf16 activations of any width and alignment -> XT bf16 terms [XT][M][Kp], zeros beyond K
template <typename T, int XT>
__global__ void __launch_bounds__(256)
stage_bf16_kernel(const T *x, size_t M, size_t K, size_t Kp, int vec_ok, uint16_t *__restrict__ terms) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t per_row = Kp >> 3, total = M * per_row, plane = M * Kp;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t m = i / per_row, c = (i % per_row) * 8;
        float v[8];
        if (vec_ok && c + 8 <= K) load_vec8<T>(x + m * K + c, v);
        else load_guarded8<T>(x + m * K + c, c < K ? K - c : 0, v);
#pragma unroll
        for (int t = 0; t < XT; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
                // truncated to bf16 (a NaN whose payload would be cut off keeps one)
                const uint32_t ha = a & 0xFFFF0000u, hb = b & 0xFFFF0000u;
                w[j] = (v[2 * j] != v[2 * j] ? 0x7FFFu : ha >> 16) | (v[2 * j + 1] != v[2 * j + 1] ? 0x7FFF0000u : hb);
                if (t + 1 < XT) {  // what is left; nothing of an infinity or a NaN
                    v[2 * j] = (a & 0x7F800000u) == 0x7F800000u ? 0.0f : v[2 * j] - __uint_as_float(ha);
                    v[2 * j + 1] = (b & 0x7F800000u) == 0x7F800000u ? 0.0f : v[2 * j + 1] - __uint_as_float(hb);
                }
            }
            *reinterpret_cast<uint4 *>(terms + t * plane + m * Kp + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

template <int TOK, int XT, bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kW4Threads, 1)
gemm_w4_bf16_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w2, const __grid_constant__ CUtensorMap tmap_x,
                    const uint8_t *__restrict__ w_pieces, const uint8_t *__restrict__ w2_pieces, Operands ops, YT *__restrict__ y, int M, int N, int K, size_t ldy,
                    int epilogue, int S, int rounds_per_cta, DeviceStatus *status) {
    using C = W4Cfg<TOK, XT, NV, GATED>;
    constexpr int kChan = GATED ? 64 : 128;
    constexpr int kMode = GATED ? kEpiLanesPaired : kEpiPlain;
    pdl_launch_dependents();
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem_raw);
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bar_area = smem + C::kStages * C::kStageBytes;
    Ctl *ctl = reinterpret_cast<Ctl *>(bar_area + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (the rank from the block's index: a value that the compiler knows to be the same in all lanes, as the operands of TMA and
    // tcgen05 instructions are that derive from it)
    const uint32_t rank = blockIdx.x % (unsigned)S;
    const int tile = (int)(blockIdx.x / (unsigned)S);
    const int m_tiles = (M + TOK - 1) / TOK;
    const int m0 = tile % m_tiles * TOK, n0 = tile / m_tiles * kChan;
    const int rounds_total = (K + kW4StageK - 1) / kW4StageK, r_begin = (int)rank * rounds_per_cta;
    const int rounds = min(rounds_total - r_begin, rounds_per_cta);  // >= 1 by construction of the grid
    const int parts = C::kLow + min(rounds, C::kLeading);            // accumulators that hold something
    const size_t pieces = (size_t)((K + 255) >> 8) * (NV ? 4 : 2);
    constexpr uint32_t kFullBar = 0, kAreadyBar = C::kStages * 8, kEmptyBar = 2 * C::kStages * 8, kAccBar = 3 * C::kStages * 8;
    const uint32_t bars = smem_u32(bar_area), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 1);
            mbar_init(bars + kAreadyBar + s * 8, 4);
            mbar_init(bars + kEmptyBar + s * 8, 1);
        }
        mbar_init(bars + kAccBar, 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        tc_alloc_512(smem_u32(&ctl->tmem_base));
        tc_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, ctl->tmem_base, 0);  // (uniform to the compiler)
    bool ok = true;

    if (warp == 0) {
        if (elect_one()) {
            auto load_w = [&](int i, int s) {
                const uint32_t dst = smem_base + s * C::kStageBytes, fb = bars + kFullBar + s * 8;
                const int r = r_begin + i;
                mbar_expect_tx(fb, C::kTxBytes);
                const size_t at = ((size_t)(n0 >> 7) * pieces + (size_t)r * C::kPieces) * 512;
                tma_load_2d(dst, &tmap_w, r * C::kCodeRow, n0, fb);
                bulk_load_1d(dst + C::kScaleOff, w_pieces + at, C::kPieces * 512, fb);
                if constexpr (GATED) {
                    tma_load_2d(dst + 64 * C::kCodeRow, &tmap_w2, r * C::kCodeRow, n0, fb);
                    bulk_load_1d(dst + C::kScaleOff + C::kPieces * 512, w2_pieces + at, C::kPieces * 512, fb);
                }
            };
            auto load_x = [&](int i, int s) {
                const uint32_t dst = smem_base + s * C::kStageBytes + C::kXOff, fb = bars + kFullBar + s * 8;
#pragma unroll
                for (int t = 0; t < XT; ++t)
#pragma unroll
                    for (int j = 0; j < kW4StageK / 64; ++j) tma_load_2d(dst + (t * (kW4StageK / 64) + j) * C::kXBox, &tmap_x, (r_begin + i) * kW4StageK + j * 64, m0 + t * M, fb);
            };
            const int pre = rounds < C::kStages ? rounds : C::kStages;
            for (int i = 0; i < pre; ++i) load_w(i, i);
            pdl_wait();
            for (int i = 0; i < pre; ++i) load_x(i, i);
            uint32_t s = 0, ph = 0;
            for (int i = pre; i < rounds; ++i) {
                if (!mbar_wait_close<kTimeoutW4>(bars + kEmptyBar + s * 8, ph, ctl, status, 0, s)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TOK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            pdl_wait();  // (as the converters)
            uint32_t s = 0, ph = 0, lead = 0;  // lead: the accumulator of this stage's leading terms
            bool good = true;
            for (int i = 0; i < rounds; ++i) {
                // (the converters have waited for the stage: its activations are there too)
                good = mbar_wait_close<kTimeoutW4>(bars + kAreadyBar + s * 8, ph, ctl, status, 2, s);
                if (!good) break;
                tc_fence_after();
                const uint64_t bdesc = make_b_desc(smem_base + s * C::kStageBytes + C::kXOff);
                const uint32_t a = tmem + C::kABase + s * C::kACols;
#pragma unroll
                for (int j = 0; j < kW4StageK / 64; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int t = 0; t < XT; ++t)
                            tc_mma_ts(tmem + (t == 0 ? C::kLow + lead : 0) * TOK, a + j * 32 + q * 8,
                                      bdesc + (uint64_t)(((t * (kW4StageK / 64) + j) * C::kXBox + q * 32) >> 4), idesc,
                                      (i >= (t == 0 ? C::kLeading : 1) || j > 0 || q > 0 || t > 1) ? 1u : 0u);
                tc_commit(bars + kEmptyBar + s * 8);  // frees the stage's shared memory and its A columns
                if (++s == C::kStages) { s = 0; ph ^= 1; }
                if (C::kLeading > 1 && ++lead == C::kLeading) lead = 0;
            }
            if (good) tc_commit(bars + kAccBar);
        }
        __syncwarp();
    } else {
        const int group = (warp - 2) >> 2, quad = warp & 3, row = quad * 32 + lane;
        // the weight row this lane widens: gated tiles alternate between the gate box (rows 0..63) and the up box (64..127)
        const int srow = GATED ? (row & 1) * 64 + (row >> 1) : row;
        const int swz = (srow >> 1) & 3;
        // its scales: row of the piece, which for a gated tile is one of 64 in the lower or upper half of a 128-row piece
        const int prow = GATED ? (n0 & 64) + (row >> 1) : row;
        const int scale_at = C::kScaleOff + (GATED ? (row & 1) * C::kPieces * 512 : 0) + (prow & 31) * 16 + (prow >> 5) * 4;
        pdl_wait();  // a stage is full only with its activations; outputs may be in use by the previous kernel
        for (int i = 0; i < rounds; ++i) {
            const int s = i % C::kStages;
            if (s % kW4Groups != group) continue;
            mbar_wait_all<kTimeoutW4>(bars + kFullBar + s * 8, (i / C::kStages) & 1, ctl, status, 3, s);
            tc_fence_after();
            const uint8_t *stage = smem + s * C::kStageBytes;
            uint32_t f[kW4StageK / 32][2];  // factors of the row's blocks
            if constexpr (NV) {
#pragma unroll
                for (int p = 0; p < kW4StageK / 64; ++p) {
                    const uint32_t w = *reinterpret_cast<const uint32_t *>(stage + scale_at + p * 512);
                    e4m3_bf16x2(w, f[2 * p][0], f[2 * p][1]);
                    e4m3_bf16x2(w >> 16, f[2 * p + 1][0], f[2 * p + 1][1]);
                }
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(stage + scale_at);
#pragma unroll
                for (int b = 0; b < kW4StageK / 32; ++b) f[b][0] = f[b][1] = e8m0_bf16x2((w >> (8 * b)) & 0xFFu);
            }
#pragma unroll
            for (int j = 0; j < kW4StageK / 64; ++j) {
                uint32_t packed[32];
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    widen32(*reinterpret_cast<const uint4 *>(stage + srow * C::kCodeRow + (((2 * j + b) ^ swz) << 4)), f[2 * j + b][0], f[2 * j + b][1], packed + 16 * b);
                tc_st32(tmem + ((uint32_t)(quad * 32) << 16) + C::kABase + s * C::kACols + j * 32, packed);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kAreadyBar + s * 8);
        }
        mbar_wait_all<kTimeoutW4>(bars + kAccBar, 0, ctl, status, 4, 0);
        ok = warp_ok(ctl);
        tc_fence_after();
        if (S == 1)
            cluster_finish<TOK, kW4Groups, kMode, YT>(tmem, smem, nullptr, 1, 0, group, quad, lane, ok, ops, y, M, N, ldy, epilogue, n0, m0, nullptr, 0, parts);
    }
    if (S > 1) {
        const int group = (warp - 2) >> 2, quad = warp & 3;
        tc_fence_before();
        __syncwarp();
        cluster_arrive();  // every CTA of the tile has its sums: the stages are idle everywhere
        cluster_wait();
        tc_fence_after();
        if (warp >= 2 && ok) cluster_send<TOK, kW4Groups, kMode>(tmem, smem_base + C::kSlotOff, S, rank, group, quad, lane, parts);
        __syncwarp();
        cluster_arrive();  // and has received the others'
        cluster_wait();
        if (warp >= 2)
            cluster_finish<TOK, kW4Groups, kMode, YT>(tmem, smem, reinterpret_cast<const float *>(smem + C::kSlotOff), S, rank, group, quad, lane, ok, ops, y, M, N,
                                                      ldy, epilogue, n0, m0, nullptr, 0, parts);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (ctl->abort_flag) {
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies and MMAs in flight get a bounded moment to land
        }
        tc_fence_after();
        __syncwarp();
        tc_dealloc_512(tmem);
    }
}

}  // namespace
}  // namespace shrewq
