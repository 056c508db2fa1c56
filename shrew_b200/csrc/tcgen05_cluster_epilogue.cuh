// Epilogue of the tcgen05 forwards over 4-bit weights: accumulators in tensor memory -> scale / bias / elementwise op -> output, with the
// k range optionally split over the CTAs of a cluster.
//
// Where the output tiles alone leave most SMs idle, a tile is computed by a cluster of S CTAs (2, 4 or 8), each over its part of k.  Their
// sums meet in shared memory: every CTA (of a narrow tile the first few: 16 tokens are the least) finishes its share of the tile's tokens
// and receives the other CTAs' raw sums of those tokens by plain stores into its pipeline stages, which are idle by then; the parts are
// added in rank order, so the result does not depend on timing.
// Against partial sums in global memory that costs no workspace (two streams, a captured graph) and no second trip through L2.
//
// A thread holds one channel (tensor-memory lane) and walks over 16 tokens at a time; values go through a [16 tokens][channels] staging
// tile so that whole token rows are stored 16 bytes a thread (element by element where rows are not on 16-byte boundaries).
//
// MODE: kEpiPlain; kEpiLanes: even lanes are gate rows, odd lanes the up rows of the same 64 channels; kEpiColumns: gate sums in columns
// [0, NCOLS), up sums of the same lanes' channels in [NCOLS, 2 NCOLS).
#pragma once

#include "ptx_cluster.cuh"
#include "ptx_fp4.cuh"
#include "ptx_tcgen05_fp4.cuh"
#include "tcgen05_common.cuh"
#include "tcgen05_epilogue.cuh"

namespace shrewq {
namespace {

// Bounded waits of the kernels whose stages take a few hundred cycles.  One thread: polls back to back for a while (mbarrier.try_wait
// suspends a thread that comes too early, and it was woken some 500 cycles after the phase completed), then as the other kernels do.
constexpr uint32_t kSpinClose = SHREWQ_SPIN_FAST_LIMIT;
template <uint32_t CODE>
__device__ __forceinline__ bool mbar_wait_close(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    for (uint32_t i = 0; i < kSpinClose; ++i)
        if (mbar_test(bar, parity)) return true;
    return mbar_wait_slow(bar, parity, ctl, st, role, stage, CODE);
}
// The same for a barrier on which the other CTA's threads arrive (mbar_arrive_release_cluster)
template <uint32_t CODE>
__device__ __forceinline__ bool mbar_wait_close_cluster(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    for (uint32_t i = 0; i < kSpinClose; ++i)
        if (mbar_test_acquire_cluster(bar, parity)) return true;
    return mbar_wait_slow(bar, parity, ctl, st, role, stage, CODE) && mbar_test_acquire_cluster(bar, parity);
}
// A whole warp: every lane looks (67 cycles where the phase is complete; one lane and a shuffle take 110, one lane, a shuffle and a second
// look by all, as mbar_wait_warp_c has it, 270).  A wait that runs out raises the abort flag and the warp goes on, so that its lanes stay
// together: what it computes then is not stored.  warp_ok() says afterwards whether anything gave up.
template <uint32_t CODE>
__device__ __forceinline__ void mbar_wait_all(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    mbar_wait_close<CODE>(bar, parity, ctl, st, role, stage);
    __syncwarp();
}
// A whole warp beside others that must not be disturbed: one lane looks, PAUSE nanoseconds apart.  A look by 32 lanes keeps the SM's
// shared-memory path busy for some 32 cycles, and 16 warps that look back to back slow every other access to it.
template <uint32_t CODE, uint32_t PAUSE>
__device__ __forceinline__ void mbar_wait_lane(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    if ((threadIdx.x & 31) == 0) {
        bool done = mbar_test(bar, parity);
        for (uint32_t i = 0; i < kSpinClose && !done; ++i) {
            if (PAUSE) __nanosleep(PAUSE);
            done = mbar_test(bar, parity);
        }
        if (!done) mbar_wait_slow(bar, parity, ctl, st, role, stage, CODE);
    }
    __syncwarp();
}
__device__ __forceinline__ bool warp_ok(Ctl *ctl) { return __all_sync(0xFFFFFFFFu, ctl->abort_flag == 0) != 0; }

enum { kEpiPlain = 0, kEpiLanesPaired = 1, kEpiColumns = 2 };
constexpr int kEpiChunk = 16;                              // tokens a step
constexpr int kEpiStageBytes = kEpiChunk * 128 * 4;        // a group's staging tile

template <int NCOLS, int MODE>
struct ClusterEpi {
    static constexpr int kAccs = MODE == kEpiColumns ? 2 : 1;
    // received sums: [source][accumulator][tokens of a finisher][128 lanes] f32 from `slots` on; this is the most (8 CTAs)
    static constexpr int kSlotBytes = kAccs * (NCOLS >= 128 ? NCOLS : 7 * kEpiChunk) * 128 * 4;
};
// CTAs of a cluster of S that finish tokens of a tile of NCOLS
template <int NCOLS>
__device__ __forceinline__ int cluster_finishers(int S) { return S < NCOLS / kEpiChunk ? S : NCOLS / kEpiChunk; }

// 16 columns of the first of `parts` accumulators, NCOLS columns apart, with the others' added in their order
template <int NCOLS>
__device__ __forceinline__ void load_sums(uint32_t taddr, int parts, uint32_t (&sum)[kEpiChunk]) {
    tc_ld16(taddr, sum);
    tc_wait_ld();
    for (int n = 1; n < parts; ++n) {
        uint32_t r[kEpiChunk];
        tc_ld16(taddr + n * NCOLS, r);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < kEpiChunk; ++j) sum[j] = __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(r[j]));
    }
}

// Sends this CTA's raw sums of the other CTAs' tokens to them.  One call per epilogue thread; the receivers' stages must be idle (a
// cluster barrier before), the sums are there after the next cluster barrier.
template <int NCOLS, int G, int MODE>
__device__ __forceinline__ void cluster_send(uint32_t tmem_d, uint32_t slots_local, int S, uint32_t rank, int group, int quad, int lane, int parts = 1) {
    const int F = cluster_finishers<NCOLS>(S), tokens = NCOLS / F, row = quad * 32 + lane;
    const uint32_t taddr = tmem_d + ((uint32_t)(quad * 32) << 16);
    const int chunks = tokens / kEpiChunk, per_dest = ClusterEpi<NCOLS, MODE>::kAccs * chunks;
    const int dests = (int)rank < F ? F - 1 : F;
    for (int i = group; i < dests * per_dest; i += G) {
        const int step = i / per_dest, acc = i % per_dest / chunks, c = i % chunks;
        const uint32_t dest = (rank + 1 + step) % F;       // everybody starts with another receiver (a finisher never meets itself)
        const uint32_t source = rank < dest ? rank : rank - 1;
        uint32_t r[kEpiChunk];
        if constexpr (ClusterEpi<NCOLS, MODE>::kAccs == 1) load_sums<NCOLS>(taddr + dest * tokens + c * kEpiChunk, parts, r);
        else {
            tc_ld16(taddr + acc * NCOLS + dest * tokens + c * kEpiChunk, r);
            tc_wait_ld();
        }
        const uint32_t at = map_to_cta(slots_local, dest) +
                            (uint32_t)((((int)source * ClusterEpi<NCOLS, MODE>::kAccs + acc) * tokens + c * kEpiChunk) * 512 + row * 4);
#pragma unroll
        for (int j = 0; j < kEpiChunk; ++j) st_cluster_u32(at + j * 512, r[j]);
    }
}

// Finishes this CTA's share of the tokens, m0 the tile's first token.  One call per epilogue thread (G groups of 128).
// TOKENS: the sums of token m are first multiplied by 2^(exps[m] + back).  parts: accumulators that a sum is kept in (one but for kEpiColumns' two).
template <int NCOLS, int G, int MODE, typename YT, bool TOKENS = false>
__device__ __forceinline__ void cluster_finish(uint32_t tmem_d, uint8_t *stage_base, const float *slots, int S, uint32_t rank, int group, int quad, int lane, bool ok,
                                               const Operands &ops, YT *__restrict__ y, int M, int N, size_t ldy, int epilogue, int n0, int m0,
                                               const int *exps = nullptr, int back = 0, int parts = 1) {
    constexpr int CW = kEpiChunk, CH = MODE == kEpiLanesPaired ? 64 : 128, RB = CH * (int)sizeof(YT), EPV = 16 / (int)sizeof(YT), PPR = RB / 16, PIECES = CW * PPR;
    constexpr int ACCS = ClusterEpi<NCOLS, MODE>::kAccs;
    const int F = cluster_finishers<NCOLS>(S), tokens = NCOLS / F, row = quad * 32 + lane;
    const uint32_t taddr = tmem_d + ((uint32_t)(quad * 32) << 16);
    const bool is_up = MODE == kEpiLanesPaired && (row & 1);
    const int ch = MODE == kEpiLanesPaired ? row >> 1 : row, n = n0 + ch;
    const bool n_ok = n < N;
    float sc[ACCS], bs[ACCS];
    sc[0] = n_ok ? (is_up ? ops.scales2 : ops.scales)[n] : 0.0f;
    const float *b0 = is_up ? ops.bias2 : ops.bias;
    bs[0] = n_ok && b0 ? b0[n] : 0.0f;
    if constexpr (ACCS == 2) {
        sc[1] = n_ok ? ops.scales2[n] : 0.0f;
        bs[1] = n_ok && ops.bias2 ? ops.bias2[n] : 0.0f;
    }
    uint8_t *stage = stage_base + group * kEpiStageBytes;
    YT *out_st = reinterpret_cast<YT *>(stage);
    const bool vec_ok = ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * sizeof(YT))) & 15) == 0;
    const int chunks = (int)rank < F ? tokens / CW : 0, first_col = (int)rank * tokens;
#pragma unroll 1
    for (int c = group; c < chunks; c += G) {
        if (ok) {
            uint32_t raw[ACCS][CW];
            if constexpr (ACCS == 1) load_sums<NCOLS>(taddr + first_col + c * CW, parts, raw[0]);
            else {
#pragma unroll
                for (int a = 0; a < ACCS; ++a) tc_ld16(taddr + a * NCOLS + first_col + c * CW, raw[a]);
                tc_wait_ld();
            }
            float v[ACCS][CW];
            if (S == 1) {
#pragma unroll
                for (int a = 0; a < ACCS; ++a)
#pragma unroll
                    for (int i = 0; i < CW; ++i) v[a][i] = __uint_as_float(raw[a][i]);
            } else {
#pragma unroll
                for (int a = 0; a < ACCS; ++a)
#pragma unroll
                    for (int i = 0; i < CW; ++i) v[a][i] = 0.0f;
                for (int z = 0; z < S; ++z) {  // in rank order
                    if (z == (int)rank) {
#pragma unroll
                        for (int a = 0; a < ACCS; ++a)
#pragma unroll
                            for (int i = 0; i < CW; ++i) v[a][i] += __uint_as_float(raw[a][i]);
                    } else {
                        const float *p = slots + (size_t)((z < (int)rank ? z : z - 1) * ACCS * tokens + c * CW) * 128 + row;
#pragma unroll
                        for (int a = 0; a < ACCS; ++a)
#pragma unroll
                            for (int i = 0; i < CW; ++i) v[a][i] += p[((size_t)a * tokens + i) * 128];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < CW; ++i) {
                if constexpr (TOKENS) {
                    const int m = m0 + first_col + c * CW + i;
                    const int e = m < M ? ld_written_s32(exps + m) + back : 0;
#pragma unroll
                    for (int a = 0; a < ACCS; ++a) v[a][i] = ldexpf(v[a][i], e);
                }
#pragma unroll
                for (int a = 0; a < ACCS; ++a) v[a][i] = v[a][i] * sc[a] + bs[a];
            }
            if constexpr (MODE == kEpiColumns) {
#pragma unroll
                for (int i = 0; i < CW; ++i) out_st[i * CH + ch] = to_out<YT>(silu_f(v[0][i]) * v[ACCS - 1][i]);
            } else if constexpr (MODE == kEpiLanesPaired) {
                // neighbouring lanes swap halves: the up lane computes the second half of the tokens, the gate lane the first
                const int keep0 = is_up ? CW / 2 : 0;
#pragma unroll
                for (int i = 0; i < CW / 2; ++i) {
                    const float other = __shfl_xor_sync(0xFFFFFFFFu, is_up ? v[0][i] : v[0][CW / 2 + i], 1);
                    const float mine = is_up ? v[0][CW / 2 + i] : v[0][i];
                    const float g = is_up ? other : mine, u = is_up ? mine : other;
                    out_st[(keep0 + i) * CH + ch] = to_out<YT>(silu_f(g) * u);
                }
            } else {
                const bool relu = epilogue == SHREWQ_EPILOGUE_RELU;
#pragma unroll
                for (int i = 0; i < CW; ++i) out_st[i * CH + ch] = to_out<YT>(relu ? relu_nan(v[0][i]) : v[0][i]);
            }
        }
        named_bar_sync(2 + group, 128);  // the staging tile is complete
        if (ok) {
            const int mc = m0 + first_col + c * CW;
            if (vec_ok) {
#pragma unroll
                for (int p = row; p < PIECES; p += 128) {
                    const int tr = p / PPR, seg = p % PPR, m = mc + tr, nn = n0 + seg * EPV;
                    if (m >= M || nn >= N) continue;
                    YT *dst = y + (size_t)m * ldy + nn;
                    if (nn + EPV <= N) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(stage + tr * RB + seg * 16);
                    else
                        for (int e = 0; e < EPV && nn + e < N; ++e) dst[e] = out_st[tr * CH + seg * EPV + e];
                }
            } else {
#pragma unroll 4
                for (int e = row; e < CW * CH; e += 128) {
                    const int tr = e / CH, cn = e % CH, m = mc + tr, nn = n0 + cn;
                    if (m < M && nn < N) y[(size_t)m * ldy + nn] = out_st[e];
                }
            }
        }
        named_bar_sync(2 + group, 128);  // the next chunk rewrites it
    }
}

}  // namespace
}  // namespace shrewq
