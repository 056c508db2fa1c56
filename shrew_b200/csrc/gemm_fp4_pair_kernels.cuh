// The 4-bit by 4-bit forward (gemm_fp4_kernels.cuh) on CTA pairs, for batches whose tiles fill the machine: clusters of two CTAs compute
// tiles of 256 weight rows by 256 tokens with tcgen05.mma.cta_group::2, one after the other.
//
// Why: a single CTA's 128 x 256 tile needs 51 KB a stage of 256 k, which at the 64 to 67 bytes a cycle that an SM takes in last 780 cycles,
// against 512 of matrix work.  In a pair each CTA brings its own 128 rows and only half of the tokens: 35 KB, 540 cycles.
//
// Each CTA holds 128 rows of A with their scales, 128 of the 256 tokens of B, and the scales of all 256 tokens; the leader issues
// tcgen05.cp and tcgen05.mma for both, and a stage is released to both CTAs (tcgen05.commit).
// GATED: even rows of A are gate rows, odd ones the up rows of the same 64 channels, so that neighbouring lanes of the accumulator hold both
// values of a channel.
//
// Warp roles: warp 0 = tensor-memory allocation, then in the leader the MMAs, in the other CTA the relay of its full stages to the leader;
// 8 epilogue warps; 8 copying warps, two groups of 4 that take the stages in turn (a group's wait for its stage and its requests take some 400
// cycles, nearly a stage).  Copies arrive on the stage's barrier by themselves (cp.async.mbarrier.arrive), and the thread that waits there
// makes them visible to the tensor core.  The relay is one plain arrival a stage: with .release.cluster, by each copying warp, it took 1200
// cycles a stage.  The copying warps run ahead into the next tile during an epilogue; the MMAs wait until the accumulators have been read.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "gemm_fp4_kernels.cuh"

namespace shrewq {
namespace {

constexpr int kPairTok = 256, kPairHalf = 128;
constexpr int kPairThreads = 32 + 256 + 256;
constexpr uint32_t kTimeoutFp4Pair = 8;  // DeviceStatus::timeout_flag of this kernel

template <bool NV, bool GATED, typename YT>
struct Fp4PairCfg {
    static constexpr int kPieces = NV ? 4 : 2;
    static constexpr int kABytes = 128 * kFp4RowBytes, kBBytes = kPairHalf * kFp4RowBytes;
    static constexpr int kSfaBytes = kPieces * 512, kSfbBytes = 2 * kPieces * 512;
    static constexpr int kBOff = kABytes, kSfaOff = kBOff + kBBytes, kSfbOff = kSfaOff + kSfaBytes, kStageBytes = kSfbOff + kSfbBytes;
    static constexpr int kAccCols = kPairTok, kSfCols = 3 * kPieces * 4;
    static constexpr int kChannels = GATED ? 64 : 128;                                  // of a CTA
    static constexpr int kOutBytes = kEpiChunk * kChannels * (int)sizeof(YT);           // a staging tile; two for each epilogue group
    static constexpr int kMaxSmem = (225 * 1024 - 4 * kOutBytes) / kStageBytes, kMaxTmem = (512 - kAccCols) / kSfCols;
    static constexpr int kStages = kMaxSmem < kMaxTmem ? kMaxSmem : kMaxTmem;
    static constexpr int kOutOff = kStages * kStageBytes, kBarOff = kOutOff + 4 * kOutBytes;
    static constexpr int kSmemBytes = kBarOff + 1024 + 1024;
    static_assert(kStages >= 4 && kSmemBytes <= 227 * 1024 && kStageBytes % 1024 == 0, "stages");
    static_assert((2 * kStages + 2) * 8 <= 512, "barriers");
};

// 16 tokens at a time of this CTA's 128 rows: sums -> scale, bias, elementwise op -> staging tile -> whole rows of y.  The tile is written
// while the one before is still being read, so one barrier a step is enough.  `step` counts them.
template <bool GATED, typename YT>
__device__ __forceinline__ void pair_epilogue(uint32_t tmem_d, uint8_t *stages, uint32_t &step, uint32_t acc_free_leader, int group, int quad, int lane, bool ok,
                                              const Operands &ops, YT *__restrict__ y, int M, int N, size_t ldy, int epilogue, int n0, int m0, bool vec_ok) {
    constexpr int CW = kEpiChunk, CH = GATED ? 64 : 128, RB = CH * (int)sizeof(YT), EPV = 16 / (int)sizeof(YT), PPR = RB / 16, PIECES = CW * PPR;
    const int row = quad * 32 + lane, ch = GATED ? row >> 1 : row, n = n0 + ch;
    const uint32_t taddr = tmem_d + ((uint32_t)(quad * 32) << 16);
    const bool is_up = GATED && (row & 1), n_ok = n < N;
    const float *bias = is_up ? ops.bias2 : ops.bias;
    const float sc = n_ok ? (is_up ? ops.scales2 : ops.scales)[n] : 0.0f, bs = n_ok && bias ? bias[n] : 0.0f;
    uint32_t raw[CW];
    tc_ld16(taddr + group * CW, raw);
#pragma unroll 1
    for (int c = group; c < kPairTok / CW; c += kFp4Groups, ++step) {
        uint8_t *stage = stages + (group * 2 + (step & 1)) * (CW * RB);
        YT *out_st = reinterpret_cast<YT *>(stage);
        tc_wait_ld();
        if constexpr (GATED) {
            // the up lane finishes the second half of the tokens, the gate lane the first
            float v[CW];
#pragma unroll
            for (int i = 0; i < CW; ++i) v[i] = __uint_as_float(raw[i]) * sc + bs;
            const int keep0 = is_up ? CW / 2 : 0;
#pragma unroll
            for (int i = 0; i < CW / 2; ++i) {
                const float other = __shfl_xor_sync(0xFFFFFFFFu, is_up ? v[i] : v[CW / 2 + i], 1), mine = is_up ? v[CW / 2 + i] : v[i];
                out_st[(keep0 + i) * CH + ch] = to_out<YT>(silu_f(is_up ? other : mine) * (is_up ? mine : other));
            }
        } else {
            const bool relu = epilogue == SHREWQ_EPILOGUE_RELU;
#pragma unroll
            for (int i = 0; i < CW; ++i) {
                const float v = __uint_as_float(raw[i]) * sc + bs;
                out_st[i * CH + ch] = to_out<YT>(relu ? fmaxf(v, 0.0f) : v);
            }
        }
        if (c + kFp4Groups < kPairTok / CW) tc_ld16(taddr + (c + kFp4Groups) * CW, raw);
        else {  // everything has been read: the next tile's MMAs may write
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_free_leader);
        }
        named_bar_sync(2 + group, 128);  // the staging tile is complete
        if (!ok) continue;
        const int mc = m0 + c * CW;
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
                const int tr = e / CH, m = mc + tr, nn = n0 + e % CH;
                if (m < M && nn < N) y[(size_t)m * ldy + nn] = out_st[e];
            }
        }
    }
}

// Grid: pairs * 2 CTAs; pair p takes the tiles p, p + pairs, ..., token tiles fastest.
template <bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_fp4_pair_kernel(const uint8_t *__restrict__ w_codes, const uint8_t *__restrict__ w2_codes, const uint8_t *__restrict__ x_codes,
                     const uint8_t *__restrict__ w_pieces, const uint8_t *__restrict__ w2_pieces, const uint8_t *__restrict__ x_pieces, Operands ops,
                     YT *__restrict__ y, int M, int N, int K, size_t ldy, int epilogue, int tiles, int pairs, DeviceStatus *status) {
    using C = Fp4PairCfg<NV, GATED, YT>;
    pdl_launch_dependents();
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem_raw);
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Ctl *ctl = reinterpret_cast<Ctl *>(smem + C::kBarOff + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1u;  // 0 = leader
    const int pair = (int)(blockIdx.x >> 1), m_tiles = (M + kPairTok - 1) / kPairTok;
    const int rounds = (K + kFp4StageK - 1) / kFp4StageK;
    const size_t pieces = (size_t)rounds * C::kPieces;
    constexpr uint32_t kFullBar = 0, kEmptyBar = C::kStages * 8, kAccFullBar = 2 * C::kStages * 8, kAccFreeBar = kAccFullBar + 8;
    const uint32_t bars = smem_u32(smem + C::kBarOff), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 128 + (rank == 0 ? 1 : 0));  // a group's copies; in the leader also the relay
            mbar_init(bars + kEmptyBar + s * 8, 1);
        }
        mbar_init(bars + kAccFullBar, 1);
        mbar_init(bars + kAccFreeBar, 2 * 4 * kFp4Groups);  // (the leader's is used)
        mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        tc_alloc_512_pair(smem_u32(&ctl->tmem_base));
        tc_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();  // both CTAs' barriers exist before anyone arrives across the pair
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, ctl->tmem_base, 0);  // (uniform to the compiler)

    if (warp == 0) {
        if (rank == 1 && elect_one()) {
            const uint32_t full_leader = map_to_cta(bars + kFullBar, 0);
            uint32_t s = 0, ph = 0;
            bool good = true;
            pdl_wait();
            for (int tile = pair; good && tile < tiles; tile += pairs)
                for (int i = 0; i < rounds; ++i) {
                    good = mbar_wait_close<kTimeoutFp4Pair>(bars + kFullBar + s * 8, ph, ctl, status, 1, s);
                    if (!good) break;
                    fence_proxy_async_smem();
                    mbar_arrive_cluster(full_leader + s * 8);
                    if (++s == C::kStages) { s = 0; ph ^= 1; }
                }
        }
        if (rank == 0 && elect_one()) {
            pdl_wait();  // a stage is full only with its activations: the time limit of the waits starts when they exist
            uint32_t s = 0, ph = 0, done = 0;
            bool good = true;
            for (int tile = pair; good && tile < tiles; tile += pairs, ++done) {
                if (done > 0 && !mbar_wait_close<kTimeoutFp4Pair>(bars + kAccFreeBar, (done - 1) & 1u, ctl, status, 3, 0)) break;
                tc_fence_after();
                for (int i = 0; i < rounds; ++i) {
                    good = mbar_wait_close<kTimeoutFp4Pair>(bars + kFullBar + s * 8, ph, ctl, status, 1, s);
                    if (!good) break;
                    fence_proxy_async_smem();
                    tc_fence_after();
                    const uint32_t base = smem_base + s * C::kStageBytes, sf = tmem + C::kAccCols + s * C::kSfCols;
                    constexpr int kSfbCol = C::kPieces * 4;
                    const uint64_t adesc = make_b_desc(base), bdesc = make_b_desc(base + C::kBOff), sdesc = make_scale_desc(base + C::kSfaOff);
#pragma unroll
                    for (int p = 0; p < C::kPieces; ++p) {
                        const uint32_t sfa = sf + p * 4, sfb = sf + kSfbCol + p * 8;
                        tc_cp_scales_pair(sfa, sdesc + (uint64_t)(p * 32));
#pragma unroll
                        for (int j = 0; j < 2; ++j) tc_cp_scales_pair(sfb + j * 4, sdesc + (uint64_t)((C::kSfaBytes >> 4) + (j * C::kPieces + p) * 32));
#pragma unroll
                        for (int h = 0; h < 4 / C::kPieces; ++h) {
                            const int q = p * (4 / C::kPieces) + h;
                            tc_mma_fp4_pair<NV>(tmem, adesc + (uint64_t)((q * 32) >> 4), bdesc + (uint64_t)((q * 32) >> 4),
                                                fp4_idesc(NV, 256, kPairTok, (uint32_t)h * 2u), sfa, sfb, (i > 0 || q > 0) ? 1u : 0u);
                        }
                    }
                    tc_commit_pair(bars + kEmptyBar + s * 8);
                    if (++s == C::kStages) { s = 0; ph ^= 1; }
                }
                if (good) tc_commit_pair(bars + kAccFullBar);
            }
        }
        __syncwarp();
    } else if (warp <= 4 * kFp4Groups) {
        // ---------------- epilogue ----------------
        const int group = (warp - 1) >> 2, quad = warp & 3;
        const uint32_t acc_free_leader = map_to_cta(bars + kAccFreeBar, 0);
        const bool vec_ok = ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * sizeof(YT))) & 15) == 0;
        uint32_t step = 0, done = 0;
        pdl_wait();  // y may be in use by the previous kernel of the stream
        for (int tile = pair; tile < tiles; tile += pairs, ++done) {
            mbar_wait_all<kTimeoutFp4Pair>(bars + kAccFullBar, done & 1u, ctl, status, 4, 0);
            const bool ok = warp_ok(ctl);
            tc_fence_after();
            pair_epilogue<GATED, YT>(tmem, smem + C::kOutOff, step, acc_free_leader, group, quad, lane, ok, ops, y, M, N, ldy, epilogue,
                                     (tile / m_tiles * 2 + (int)rank) * C::kChannels, tile % m_tiles * kPairTok, vec_ok);
        }
    } else {
        // ---------------- copies: 16 bytes a lane, swizzled as they land ----------------
        constexpr int kInstr = 8;  // 4 rows each, of a warp: 32 rows of A, 32 of B
        const int copier = warp - 1 - 4 * kFp4Groups, cgroup = copier >> 2, cw = copier & 3, t = cw * 32 + lane;
        const size_t pitch = (size_t)((K + 31) >> 5) * 16;
        const int seg = (lane & 7) * 16, last_tile = (M - 1) >> 7;
        const uint8_t *wsrc[kInstr], *xsrc[kInstr], *sfa_src[C::kPieces], *sfb_src[2 * C::kPieces / 4];
        uint32_t at[kInstr];
#pragma unroll
        for (int j = 0; j < kInstr; ++j) {
            const int r = (cw * kInstr + j) * 4 + (lane >> 3);
            at[j] = (uint32_t)(r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        }
        auto begin = [&](int tile) {
            const int n0 = (tile / m_tiles * 2 + (int)rank) * C::kChannels, m0 = tile % m_tiles * kPairTok;
#pragma unroll
            for (int j = 0; j < kInstr; ++j) {
                const int r = (cw * kInstr + j) * 4 + (lane >> 3);
                const int n = n0 + (GATED ? r >> 1 : r), m = m0 + (int)rank * kPairHalf + r;
                wsrc[j] = (GATED && (r & 1) ? w2_codes : w_codes) + (size_t)(n < N ? n : N - 1) * pitch + seg;
                xsrc[j] = x_codes + (size_t)(m < M ? m : M - 1) * pitch + seg;
            }
            if constexpr (GATED) {  // four bytes (a row's scales) at a time: gate and up rows are interleaved
                const int r = (t & 3) * 32 + (t >> 2), n = n0 + (r >> 1) < N ? n0 + (r >> 1) : N - 1;
#pragma unroll
                for (int p = 0; p < C::kPieces; ++p)
                    sfa_src[p] = (r & 1 ? w2_pieces : w_pieces) + ((size_t)(n >> 7) * pieces + p) * 512 + (n & 31) * 16 + ((n & 127) >> 5) * 4;
            } else {
                const int wt = (n0 < N ? n0 : N - 1) >> 7;  // (rows past the end: any scales)
                sfa_src[0] = w_pieces + (size_t)wt * pieces * 512 + t * 16;
            }
#pragma unroll
            for (int j = 0; j < 2 * C::kPieces / 4; ++j) {
                const int c = j * 128 + t, half = c / (C::kPieces * 32), xt = (m0 >> 7) + half < last_tile ? (m0 >> 7) + half : last_tile;
                sfb_src[j] = x_pieces + (size_t)xt * pieces * 512 + (c % (C::kPieces * 32)) * 16;
            }
        };
        auto copy_w = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t byte = (size_t)i * kFp4RowBytes, sf = (size_t)i * C::kPieces * 512;
            const bool in = byte + seg < pitch;  // (codes past the end of a row: zeros)
#pragma unroll
            for (int j = 0; j < kInstr; ++j) copy_async_16(dst + at[j], in ? wsrc[j] + byte : wsrc[j], in);
            if constexpr (GATED) {
#pragma unroll
                for (int p = 0; p < C::kPieces; ++p) copy_async_4(dst + C::kSfaOff + p * 512 + t * 4, sfa_src[p] + sf, true);
            } else {
                if (t < C::kSfaBytes / 16) copy_async_16(dst + C::kSfaOff + t * 16, sfa_src[0] + sf, true);
            }
        };
        auto copy_x = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t byte = (size_t)i * kFp4RowBytes, sf = (size_t)i * C::kPieces * 512;
            const bool in = byte + seg < pitch;
#pragma unroll
            for (int j = 0; j < kInstr; ++j) copy_async_16(dst + C::kBOff + at[j], in ? xsrc[j] + byte : xsrc[j], in);
#pragma unroll
            for (int j = 0; j < 2 * C::kPieces / 4; ++j) copy_async_16(dst + C::kSfbOff + (j * 128 + t) * 16, sfb_src[j] + sf, true);
        };
        begin(pair);
        const int pre = rounds < C::kStages ? rounds : C::kStages;
        for (int i = cgroup; i < pre; i += 2) copy_w(i, i);
        pdl_wait();
        int it = 0;  // stages so far, of both groups
        uint32_t s = 0, ph = 0;
        for (int tile = pair; tile < tiles; tile += pairs) {
            if (it > 0) begin(tile);
            for (int i = 0; i < rounds; ++i, ++it) {
                if ((it & 1) == cgroup) {
                    if (it >= C::kStages) mbar_wait_all<kTimeoutFp4Pair>(bars + kEmptyBar + s * 8, ph ^ 1u, ctl, status, 0, s);
                    if (it >= pre) copy_w(i, s);
                    copy_x(i, s);
                    copy_async_arrive(bars + kFullBar + s * 8);
                }
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        }
    }

    // both CTAs are done with tensor memory, and with each other, before it is freed
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == 0) {
        if (ctl->abort_flag) {
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // MMAs in flight get a bounded moment to land
        }
        tc_fence_after();
        __syncwarp();
        tc_dealloc_512_pair(tmem);
    }
}

}  // namespace
}  // namespace shrewq
