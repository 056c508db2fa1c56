// Forward of a layer whose weights and activations are both 4-bit microscaled codes, on the block-scaled tensor cores (tcgen05.mma
// kind::mxf4 and kind::mxf4nvf4), sm_100a only.
//
//   y[m,n] = epi( alpha[n] * sum_k (w code * w scale)[n,k] (x code * x scale)[m,k] + bias[n] ),  f32 sums
//
// Mapping.  D[128 x TOK] += A[128 x 64] * B[TOK x 64]^T for each instruction: A = 128 weight rows, B = a tile of tokens, both packed codes in
// shared memory (TMA, 128-byte swizzle, K-major: one row of a stage is 256 codes = 128 bytes), D = f32 accumulators in tensor memory
// (lane = output channel, column = token).  The scales of a stage come as the 512-byte pieces that the quantizer and the handle lay out
// (scale_piece_offset), by 1-D bulk copies, and go to tensor memory with tcgen05.cp just ahead of the MMAs that use them; every stage
// of the ring has its own columns for them, so the release of the stage covers them too.
//
// GATED: two MMAs into two accumulators: gate rows and up rows of the same 128 channels against the same token tile; a lane then
// holds both values of its channel and the epilogue writes silu(gate) * up without an exchange.
//
// Warp roles: warp 0 = TMA producer, warp 1 = tensor-memory allocation and MMA issue, then 8 epilogue warps.  full[s] (bytes landed) ->
// MMA -> empty[s] (tcgen05.commit) -> producer; every wait is bounded as in the other tcgen05 kernels.
// Programmatic dependent launch: weights of the first stages are requested before the wait for the previous kernel, the activations'
// codes (the quantizer's output) after it.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "../../include/shrewq.h"
#include "dests.cuh"
#include "ptx_small.cuh"
#include "ptx_tcgen05.cuh"
#include "ptx_tcgen05_fp4.cuh"
#include "tcgen05_common.cuh"
#include "tcgen05_epilogue.cuh"

namespace shrewq {
namespace {

constexpr int kFp4StageK = 256;       // codes of k a stage: rows of 128 bytes
constexpr int kFp4RowBytes = 128;
constexpr int kFp4Groups = 2;         // epilogue groups of 4 warps
constexpr int kFp4GemmThreads = 64 + 128 * kFp4Groups;
constexpr uint32_t kTimeoutFp4 = 5;   // DeviceStatus::timeout_flag of this kernel

template <int TOK, bool NV, bool GATED>
struct Fp4Cfg {
    static constexpr int kMats = GATED ? 2 : 1;
    static constexpr int kPieces = NV ? 4 : 2;                            // scale pieces of 128 rows a stage
    static constexpr int kABytes = 128 * kFp4RowBytes;                     // one weight tile
    static constexpr int kBBytes = TOK * kFp4RowBytes;
    static constexpr int kTokTiles = (TOK + 127) / 128;                    // pieces' row groups of the token tile
    static constexpr int kSfaBytes = kPieces * 512, kSfbBytes = kTokTiles * kPieces * 512;
    static constexpr int kBOff = kMats * kABytes, kSfaOff = kBOff + kBBytes, kSfbOff = kSfaOff + kMats * kSfaBytes;
    static constexpr int kStageBytes = kSfbOff + kSfbBytes;
    static constexpr int kAccCols = kMats * TOK;
    static constexpr int kSfCols = (kMats + kTokTiles) * kPieces * 4;      // tensor-memory columns of a stage's scales
    static constexpr int kMaxStagesSmem = (220 * 1024) / kStageBytes;
    static constexpr int kMaxStagesTmem = (512 - kAccCols) / kSfCols;
    static constexpr int kStagesRaw = kMaxStagesSmem < kMaxStagesTmem ? kMaxStagesSmem : kMaxStagesTmem;
    static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
    static constexpr int kSmemBytes = kStages * kStageBytes + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static constexpr int kSmemRequest = kSmemBytes > 120 * 1024 ? kSmemBytes : 120 * 1024;  // one CTA an SM: it takes all of tensor memory
    static_assert(kStages >= 3 && kSmemRequest <= 227 * 1024, "stages");
    static_assert(kStageBytes % 1024 == 0 && kBOff % 1024 == 0, "tiles keep the 1024-byte swizzle alignment");
    static_assert(kStages * kStageBytes >= kFp4Groups * kEpiGroupBytes, "the epilogue's staging tiles reuse the stages");
};

__device__ __forceinline__ bool fp4_wait(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    return mbar_wait_c<kTimeoutFp4>(bar, parity, ctl, st, role, stage);
}

// Shared-memory descriptor of a scale piece: no swizzle, rows of 16 bytes, 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}

// Instruction descriptor of the block-scaled kinds: E2M1 operands (1 in both format fields), K-major, N, scale type (E8M0: bit 23), M; `sf`:
// which of a column's four scale bytes are meant, for both operands (0, or 2 for the second half of an MX piece)
__device__ __forceinline__ constexpr uint32_t fp4_idesc(bool nv, int m, int n, uint32_t sf) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (nv ? 0u : 1u << 23) | ((uint32_t)(m >> 4) << 24) | (sf << 4) | (sf << 29);
}

// silu(gate) * up from two accumulators side by side in tensor memory (gate in columns [0, NCOLS), up in [NCOLS, 2 NCOLS)); otherwise the
// staging, stores and barriers of epilogue_tile
template <int NCOLS, int G, typename YT>
__device__ __forceinline__ void epilogue_gated_columns(uint32_t tmem_d, uint8_t *stage_base, int group, int quad, int lane, bool ok, const Operands &ops,
                                                       YT *__restrict__ y, int M, int N, size_t ldy, int n0, int m0) {
    constexpr int CW = 16, CH = kEpiLanes, RB = CH * (int)sizeof(YT), EPV = 16 / (int)sizeof(YT), PPR = RB / 16, PIECES = CW * PPR;
    const int row = quad * 32 + lane, n = n0 + row;
    const uint32_t taddr = tmem_d + ((uint32_t)(quad * 32) << 16);
    const bool n_ok = n < N;
    const float sg = n_ok ? ops.scales[n] : 0.0f, su = n_ok ? ops.scales2[n] : 0.0f;
    const float bg = n_ok && ops.bias ? ops.bias[n] : 0.0f, bu = n_ok && ops.bias2 ? ops.bias2[n] : 0.0f;
    uint8_t *stage = stage_base + group * kEpiGroupBytes;
    YT *out_st = reinterpret_cast<YT *>(stage);
    const bool vec_ok = ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * sizeof(YT))) & 15) == 0;
#pragma unroll 1
    for (int c = group; c < NCOLS / CW; c += G) {
        if (ok) {
            uint32_t rg[CW], ru[CW];
            tc_ld16(taddr + c * CW, rg);
            tc_ld16(taddr + NCOLS + c * CW, ru);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < CW; ++i) {
                const float g = __uint_as_float(rg[i]) * sg + bg, u = __uint_as_float(ru[i]) * su + bu;
                out_st[i * CH + row] = to_out<YT>(silu_f(g) * u);
            }
        }
        named_bar_sync(2 + group, 128);
        if (ok) {
            for (int p = row; p < PIECES; p += 128) {
                const int tr = p / PPR, seg = p % PPR, m = m0 + c * CW + tr, nn = n0 + seg * EPV;
                if (m >= M || nn >= N) continue;
                YT *dst = y + (size_t)m * ldy + nn;
                if (vec_ok && nn + EPV <= N) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(stage + tr * RB + seg * 16);
                else
                    for (int e = 0; e < EPV && nn + e < N; ++e) dst[e] = out_st[tr * CH + seg * EPV + e];
            }
        }
        named_bar_sync(2 + group, 128);
    }
}

template <int TOK, bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kFp4GemmThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w2, const __grid_constant__ CUtensorMap tmap_x,
                const uint8_t *__restrict__ w_pieces, const uint8_t *__restrict__ w2_pieces, const uint8_t *__restrict__ x_pieces, Operands ops,
                YT *__restrict__ y, int M, int N, int K, size_t ldy, int epilogue, DeviceStatus *status) {
    using C = Fp4Cfg<TOK, NV, GATED>;
    pdl_launch_dependents();
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem_raw);
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bar_area = smem + C::kStages * C::kStageBytes;
    Ctl *ctl = reinterpret_cast<Ctl *>(bar_area + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // token tiles fastest: the CTAs that share a weight tile start together, so it comes from DRAM once
    const int m_tiles = (M + TOK - 1) / TOK;
    const int m0 = (int)(blockIdx.x % m_tiles) * TOK, n0 = (int)(blockIdx.x / m_tiles) * 128;
    const int rounds = (K + kFp4StageK - 1) / kFp4StageK;
    const size_t pieces = (size_t)rounds * C::kPieces;  // along a row
    constexpr uint32_t kFullBar = 0, kEmptyBar = C::kStages * 8, kAccBar = 2 * C::kStages * 8;
    const uint32_t bars = smem_u32(bar_area), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        ctl->tmem_base = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 1);
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
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        if (elect_one()) {
            auto load_w = [&](int i, int s) {
                const uint32_t dst = smem_base + s * C::kStageBytes, fb = bars + kFullBar + s * 8;
                mbar_expect_tx(fb, C::kStageBytes);
                const size_t at = ((size_t)(n0 >> 7) * pieces + (size_t)i * C::kPieces) * 512;
                tma_load_2d(dst, &tmap_w, i * kFp4RowBytes, n0, fb);
                bulk_load_1d(dst + C::kSfaOff, w_pieces + at, C::kSfaBytes, fb);
                if constexpr (GATED) {
                    tma_load_2d(dst + C::kABytes, &tmap_w2, i * kFp4RowBytes, n0, fb);
                    bulk_load_1d(dst + C::kSfaOff + C::kSfaBytes, w2_pieces + at, C::kSfaBytes, fb);
                }
            };
            // the token tiles of the pieces beyond the last one are read from it again: their columns are not stored
            const int last_tile = (M - 1) >> 7;
            auto load_x = [&](int i, int s) {
                const uint32_t dst = smem_base + s * C::kStageBytes, fb = bars + kFullBar + s * 8;
                tma_load_2d(dst + C::kBOff, &tmap_x, i * kFp4RowBytes, m0, fb);
#pragma unroll
                for (int j = 0; j < C::kTokTiles; ++j) {
                    const int tile = (m0 >> 7) + j < last_tile ? (m0 >> 7) + j : last_tile;
                    bulk_load_1d(dst + C::kSfbOff + j * C::kPieces * 512, x_pieces + ((size_t)tile * pieces + (size_t)i * C::kPieces) * 512, C::kPieces * 512, fb);
                }
            };
            const int pre = rounds < C::kStages ? rounds : C::kStages;
            for (int i = 0; i < pre; ++i) load_w(i, i);
            pdl_wait();
            for (int i = 0; i < pre; ++i) load_x(i, i);
            uint32_t s = 0, ph = 0;
            for (int i = pre; i < rounds; ++i) {
                if (!fp4_wait(bars + kEmptyBar + s * 8, ph, ctl, status, 0, s)) break;
                load_w(i, s);
                load_x(i, s);
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            pdl_wait();  // a stage is full only with its activations: the time limit of the waits starts when they exist
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (int i = 0; i < rounds; ++i) {
                ok = fp4_wait(bars + kFullBar + s * 8, ph, ctl, status, 1, s);
                if (!ok) break;
                tc_fence_after();
                const uint32_t base = smem_base + s * C::kStageBytes;
                const uint32_t sf = tmem + C::kAccCols + s * C::kSfCols;             // A pieces (gate, up), then B pieces
                constexpr int kSfbCol = C::kMats * C::kPieces * 4, kBStep = 4 * C::kTokTiles;
#pragma unroll
                for (int p = 0; p < C::kPieces; ++p) {
#pragma unroll
                    for (int a = 0; a < C::kMats; ++a)
                        tc_cp_scales(sf + (a * C::kPieces + p) * 4, make_scale_desc(base + C::kSfaOff + (a * C::kPieces + p) * 512));
#pragma unroll
                    for (int j = 0; j < C::kTokTiles; ++j)
                        tc_cp_scales(sf + kSfbCol + p * kBStep + j * 4, make_scale_desc(base + C::kSfbOff + (j * C::kPieces + p) * 512));
                }
                const uint64_t adesc = make_b_desc(base), bdesc = make_b_desc(base + C::kBOff);
                const uint32_t tok_col = TOK < 128 ? (uint32_t)((m0 & 127) >> 5) : 0u;  // a token tile of half a piece
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // 64 codes = 32 bytes of a row
                    constexpr bool nv = NV;
                    const int p = nv ? q : q >> 1;
                    const uint32_t idesc = fp4_idesc(nv, 128, TOK, nv ? 0u : (uint32_t)(q & 1) * 2u);
#pragma unroll
                    for (int a = 0; a < C::kMats; ++a)
                        tc_mma_fp4<NV>(tmem + a * TOK, adesc + (uint64_t)((a * C::kABytes + q * 32) >> 4), bdesc + (uint64_t)((q * 32) >> 4), idesc,
                                       sf + (a * C::kPieces + p) * 4, sf + kSfbCol + p * kBStep + tok_col, (i > 0 || q > 0) ? 1u : 0u);
                }
                tc_commit(bars + kEmptyBar + s * 8);
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
            if (ok) tc_commit(bars + kAccBar);
        }
        __syncwarp();
    } else {
        const int group = (warp - 2) >> 2, quad = warp & 3;
        pdl_wait();  // y may be in use by the previous kernel of the stream
        const bool ok = mbar_wait_warp_c<kTimeoutFp4>(bars + kAccBar, 0, ctl, status, 4, 0);
        if (ok) tc_fence_after();
        if constexpr (GATED)
            epilogue_gated_columns<TOK, kFp4Groups, YT>(tmem, smem, group, quad, lane, ok, ops, y, M, N, ldy, n0, m0);
        else
            epilogue_tile<TOK, kFp4Groups, false, YT>(tmem, smem, group, quad, lane, ok, ops, y, Dests{{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr}, 0},
                                                      M, N, ldy, epilogue, n0, m0, PartialSums{nullptr, 0, 0});
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
