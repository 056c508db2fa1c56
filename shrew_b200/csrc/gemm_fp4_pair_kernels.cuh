// The 4-bit by 4-bit forward (gemm_fp4_kernels.cuh) on CTA pairs, for batches whose tiles fill the machine: clusters of two CTAs compute
// tiles of 256 tokens by 256 weight rows with tcgen05.mma.cta_group::2, one after the other.
//
// Why: a single CTA's 128 x 256 tile needs 51 KB a stage of 256 k, which at the 64 to 67 bytes a cycle that an SM takes in last 780 cycles,
// against 512 of matrix work.  In a pair each CTA brings its own 128 tokens and only half of the weight rows: 35 KB (MX) or 38 KB (NV).
//
// A = tokens (128 in each CTA, with their scales), B = weight rows (128 in each CTA; the scales of all 256 in both); the leader issues
// tcgen05.cp and tcgen05.mma for both, and a stage is released to both CTAs (tcgen05.commit).  GATED: the first CTA brings gate rows, the
// second one the up rows of the same 128 channels.
// Tokens are the lanes of the accumulator, so a thread holds neighbouring channels of one token, gate and up values alike: it packs 16
// bytes of output at a time, and a warp turns its 32 x 32 piece into whole rows through 2 KB (4 KB for f32) of its own.  With channels as lanes, as the kernels for few
// tokens have them, every output was a two-byte store to shared memory and gate and up values had to change lanes: some 370 instructions
// for each warp and 16 columns, 7500 to 8400 cycles a tile, in which the tensor cores stood still.
//
// Warp roles: warp 0 = tensor-memory allocation, and in the leader the MMAs; four groups of 4 warps = epilogue, the first two of them also
// copies, taking the stages in turn; the last warp = relay.  Copies arrive on the stage's barrier by themselves
// (cp.async.mbarrier.arrive); the relay of each CTA waits there, makes them visible to the tensor core (fence.proxy.async) and arrives at
// the leader, publishing them to the cluster (a fence for shared memory alone: with .release.cluster the relays' arrivals held the pair up, 165 us
// instead of 117 for 4096 x 11008 with 4096 tokens, and by the copying warps, with copies in flight, they took 1200 cycles a stage).
// The accumulators, 256 columns, and the stages' scales fill tensor memory, so the MMAs of the next tile wait until the sums have been read: all
// warps that are free then take part, after the next tile's first stages are under way.
// Measured: 4096 x 11008 MX, 4096 tokens: 85 us of 116 to 118 for the call (quantizing the tokens is the rest; 3.1 PFLOP/s over all, at 1680 MHz under
// the power limit); gated 11008 x 4096 NV, 512 tokens: 35 us, 38.5 to 39.5 for the call.  A stage takes 540 to 600 cycles to bring for 512 of matrix
// work, and 256 (172) tiles for 74 pairs are 3.5 (2.3) rounds that take 4 (3): together 66 and 25 us.  The rest is most likely the MMAs' wait for
// the copying groups, which bring 4 or 5 stages of the next tile and are then in the epilogue of this one.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "gemm_fp4_kernels.cuh"

namespace shrewq {
namespace {

constexpr int kPairTok = 256, kPairHalf = 128;  // tokens of a tile, and those that a CTA brings
constexpr int kPairGroups = 4;                  // groups of 4 warps: two run the epilogue only, two also copy
constexpr int kPairThreads = 32 + 128 * kPairGroups + 32;
constexpr uint32_t kTimeoutFp4Pair = 8;  // DeviceStatus::timeout_flag of this kernel

template <bool NV, bool GATED, typename YT>
struct Fp4PairCfg {
    static constexpr int kPieces = NV ? 4 : 2;
    static constexpr int kABytes = 128 * kFp4RowBytes, kBBytes = kPairHalf * kFp4RowBytes;
    static constexpr int kSfaBytes = kPieces * 512, kSfbBytes = 2 * kPieces * 512;
    static constexpr int kBOff = kABytes, kSfaOff = kBOff + kBBytes, kSfbOff = kSfaOff + kSfaBytes, kStageBytes = kSfbOff + kSfbBytes;
    static constexpr int kSfCols = 3 * kPieces * 4;                                     // tensor memory: accumulators, then the stages' scales
    static constexpr int kChannels = GATED ? 128 : 256;                                 // of a tile
    static constexpr int kOutBytes = 32 * 32 * (int)sizeof(YT) + 512;                   // of a warp: a piece of the output, its columns' factors
    static constexpr int kMaxSmem = (225 * 1024 - 4 * kPairGroups * kOutBytes) / kStageBytes, kMaxTmem = (512 - kPairTok) / kSfCols;
    static constexpr int kStages = kMaxSmem < kMaxTmem ? kMaxSmem : kMaxTmem;
    static constexpr int kOutOff = kStages * kStageBytes, kBarOff = kOutOff + 4 * kPairGroups * kOutBytes;
    static constexpr int kSmemBytes = kBarOff + 1024 + 1024;
    static_assert(kStages >= 4 && kSmemBytes <= 227 * 1024 && kStageBytes % 1024 == 0, "stages");
    static_assert((3 * kStages + 2) * 8 <= 512, "barriers");
};

// silu(g) * u = u g / (1 + 2^(-g log2 e)), by the approximate 2^x and 1 / x (results below 2^-126 are 0, within 2^-126 |u g| of theirs): four
// instructions less than through __expf and __fdividef
__device__ __forceinline__ float pair_silu(float g, float u) {
    return g * recip_approx(1.0f + exp2_approx(-1.44269504f * g)) * u;
}

// This warp's 32 tokens: sums -> scale, bias, elementwise op -> rows of y.  Two steps of 32 sums a thread: 32 channels each (group, and 4 groups further),
// or the gate and up sums of 16.  The second step's sums are read before the first one's rows are written, so that the next tile's MMAs
// can begin.
template <bool GATED, typename YT>
struct PairEpilogue {
    static constexpr int EPV = 16 / (int)sizeof(YT), SEGS = 32 / EPV;  // 16-byte pieces of a row of 32 channels
    uint8_t *own;                                                       // [32 tokens][32 channels] of outputs, then the channels' factors
    int group, quad, lane;

    // piece j of row r, so that neither writing a piece of every row nor reading whole rows meets a bank twice
    __device__ __forceinline__ uint8_t *at(int r, int j) const { return own + (r * SEGS + (j ^ (SEGS == 8 ? r & 7 : (r >> 1) & 3))) * 16; }
    __device__ __forceinline__ float *factors() const { return reinterpret_cast<float *>(own + 32 * 32 * sizeof(YT)); }

    // scale and bias of this warp's channels: asked for before the sums are waited for
    __device__ __forceinline__ void begin(const Operands &ops, int n0, int N) const {
        float4 f;
        const int n = n0 + group * 32 + lane, n2 = GATED ? n : n + 128;
        const float *scales2 = GATED ? ops.scales2 : ops.scales, *bias2 = GATED ? ops.bias2 : ops.bias;
        f.x = n < N ? ops.scales[n] : 0.0f, f.y = n < N && ops.bias ? ops.bias[n] : 0.0f;
        f.z = n2 < N ? scales2[n2] : 0.0f, f.w = n2 < N && bias2 ? bias2[n2] : 0.0f;
        __syncwarp();  // the tile before has read its factors
        if constexpr (GATED) reinterpret_cast<float4 *>(factors())[lane] = f;
        else {
            reinterpret_cast<float2 *>(factors())[lane] = float2{f.x, f.y};
            reinterpret_cast<float2 *>(factors())[32 + lane] = float2{f.z, f.w};
        }
        __syncwarp();
    }
    __device__ __forceinline__ void load(uint32_t tmem_d, int step, uint32_t (&lo)[16], uint32_t (&hi)[16]) const {
        const uint32_t at0 = tmem_d + ((uint32_t)(quad * 32) << 16) + (GATED ? group * 32 + step * 16 : step * 128 + group * 32);
        tc_ld16(at0, lo);
        tc_ld16(at0 + (GATED ? 128 : 16), hi);
        tc_wait_ld();
    }
    __device__ __forceinline__ void pack(int first_piece, const float (&v)[16]) const {
#pragma unroll
        for (int j = 0; j < 16 / EPV; ++j) {
            union { uint4 q; YT e[EPV]; } o;
#pragma unroll
            for (int e = 0; e < EPV; ++e) o.e[e] = to_out<YT>(v[j * EPV + e]);
            *reinterpret_cast<uint4 *>(at(lane, first_piece + j)) = o.q;
        }
    }
    __device__ __forceinline__ void compute(int step, const uint32_t (&lo)[16], const uint32_t (&hi)[16], bool relu) const {
        float v[16];
        if constexpr (GATED) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float4 f = reinterpret_cast<const float4 *>(factors())[step * 16 + i];
                v[i] = pair_silu(__uint_as_float(lo[i]) * f.x + f.y, __uint_as_float(hi[i]) * f.z + f.w);
            }
            pack(step * (16 / EPV), v);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) {  // two channels' factors at a time
                    const float4 f = reinterpret_cast<const float4 *>(factors())[step * 16 + h * 8 + i / 2];
                    v[i] = __uint_as_float(h ? hi[i] : lo[i]) * f.x + f.y;
                    v[i + 1] = __uint_as_float(h ? hi[i + 1] : lo[i + 1]) * f.z + f.w;
                }
                if (relu) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = relu_nan(v[i]);
                }
                pack(h * (16 / EPV), v);
            }
        }
    }
    __device__ __forceinline__ void store(YT *__restrict__ y, int M, int N, size_t ldy, int n, int m0, bool vec_ok) const {
        __syncwarp();
#pragma unroll
        for (int p = 0; p < SEGS; ++p) {
            const int r = p * (32 / SEGS) + lane / SEGS, j = lane % SEGS, m = m0 + quad * 32 + r, nn = n + j * EPV;
            if (m >= M || nn >= N) continue;
            YT *dst = y + (size_t)m * ldy + nn;
            union { uint4 q; YT e[EPV]; } o;
            o.q = *reinterpret_cast<const uint4 *>(at(r, j));
            if (vec_ok && nn + EPV <= N) *reinterpret_cast<uint4 *>(dst) = o.q;
            else {
#pragma unroll
                for (int e = 0; e < EPV; ++e)
                    if (nn + e < N) dst[e] = o.e[e];
            }
        }
        __syncwarp();
    }
};

// Grid: pairs * 2 CTAs; pair p takes the tiles p, p + pairs, ..., token tiles fastest.
template <bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_fp4_pair_kernel(const uint8_t *__restrict__ w_codes, const uint8_t *__restrict__ w2_codes, const uint8_t *x_codes,
                     const uint8_t *__restrict__ w_pieces, const uint8_t *__restrict__ w2_pieces, const uint8_t *x_pieces, Operands ops,
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
    constexpr uint32_t kFullBar = 0, kEmptyBar = C::kStages * 8, kAccFullBar = 2 * C::kStages * 8, kAccFreeBar = kAccFullBar + 8, kReadyBar = kAccFreeBar + 8;
    const uint32_t bars = smem_u32(smem + C::kBarOff), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 128);  // a group's copies
            mbar_init(bars + kReadyBar + s * 8, 2);   // the relays (the leader's are used)
            mbar_init(bars + kEmptyBar + s * 8, 1);
        }
        mbar_init(bars + kAccFullBar, 1);
        mbar_init(bars + kAccFreeBar, 2 * 4 * kPairGroups);  // (the leader's is used)
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
        if (rank == 0 && elect_one()) {
            pdl_wait();  // a stage is full only with its activations: the time limit of the waits starts when they exist
            uint32_t s = 0, ph = 0, done = 0;
            bool good = true, ready = false;
            for (int tile = pair; good && tile < tiles; tile += pairs, ++done) {
                if (done > 0 && !mbar_wait_close<kTimeoutFp4Pair>(bars + kAccFreeBar, (done - 1) & 1u, ctl, status, 3, 0)) break;
                for (int i = 0; i < rounds; ++i) {
                    good = ready || mbar_wait_close_cluster<kTimeoutFp4Pair>(bars + kReadyBar + s * 8, ph, ctl, status, 1, s);
                    if (!good) break;
                    tc_fence_after();
                    // (a look takes 150 to 300 cycles here: the next stage's is under way while this one's MMAs are issued)
                    const uint32_t next = s + 1 == C::kStages ? 0 : s + 1, next_ph = s + 1 == C::kStages ? ph ^ 1u : ph;
                    ready = mbar_test_acquire_cluster(bars + kReadyBar + next * 8, next_ph);
                    const uint32_t base = smem_base + s * C::kStageBytes, sf = tmem + kPairTok + s * C::kSfCols;
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
                    s = next, ph = next_ph;
                }
                if (good) tc_commit_pair(bars + kAccFullBar);
            }
        }
        __syncwarp();
    } else if (warp == kPairThreads / 32 - 1) {
        // ---------------- relay: copies that have landed -> visible to the tensor core -> the leader ----------------
        if (elect_one()) {
            const uint32_t ready_leader = map_to_cta(bars + kReadyBar, 0);
            uint32_t s = 0, ph = 0;
            bool good = true;
            pdl_wait();
            for (int tile = pair; good && tile < tiles; tile += pairs)
                for (int i = 0; i < rounds; ++i) {
                    good = mbar_wait_close<kTimeoutFp4Pair>(bars + kFullBar + s * 8, ph, ctl, status, 5, s);
                    if (!good) break;
                    fence_proxy_async_smem();
                    mbar_arrive_release_cluster(ready_leader + s * 8);
                    if (++s == C::kStages) { s = 0; ph ^= 1; }
                }
        }
        __syncwarp();
    } else {
        const int group = (warp - 1) >> 2, quad = warp & 3;
        const uint32_t acc_free_leader = map_to_cta(bars + kAccFreeBar, 0);
        const bool vec_ok = ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(ldy * sizeof(YT))) & 15) == 0;
        uint32_t done = 0;
        const PairEpilogue<GATED, YT> epi{smem + C::kOutOff + (warp - 1) * C::kOutBytes, group, quad, lane};
        const bool relu = epilogue == SHREWQ_EPILOGUE_RELU;
        auto finish = [&](int tile) {
            const int n0 = tile / m_tiles * C::kChannels, m0 = tile % m_tiles * kPairTok + (int)rank * kPairHalf;
            epi.begin(ops, n0, N);
            mbar_wait_lane<kTimeoutFp4Pair, 40>(bars + kAccFullBar, done & 1u, ctl, status, 4, 0);
            ++done;
            const bool ok = warp_ok(ctl);
            tc_fence_after();
            uint32_t lo[16], hi[16];
            epi.load(tmem, 0, lo, hi);
            epi.compute(0, lo, hi, relu);
            epi.load(tmem, 1, lo, hi);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_free_leader);  // everything has been read: the next tile's MMAs may write
            if (!GATED && ok) epi.store(y, M, N, ldy, n0 + group * 32, m0, vec_ok);
            epi.compute(1, lo, hi, relu);
            if (ok) epi.store(y, M, N, ldy, n0 + group * 32 + (GATED ? 0 : 128), m0, vec_ok);
        };
        if (group >= 2) {
            pdl_wait();  // y may be in use by the previous kernel of the stream
            for (int tile = pair; tile < tiles; tile += pairs) finish(tile);
        } else {
        // ---------------- copies: 16 bytes a lane, swizzled as they land ----------------
        constexpr int kInstr = 8;  // of a warp, 4 rows each: 32 rows of each operand
        const int cw = (warp - 1) & 3, t = cw * 32 + lane;
        const uint32_t pitch = (uint32_t)((K + 31) >> 5) * 16;
        const uint32_t seg = (lane & 7) * 16, last_m = (M - 1) >> 7, last_n = (N - 1) >> 7;
        const uint8_t *wrows = GATED && rank ? w2_codes : w_codes, *wtile, *xtile, *sfw_src[C::kPieces / 2], *sfx_src;
        int w_last = 0, x_last = 0;  // last rows of the tile that there are
        // 16 bytes a lane of 4 rows at a time; the swizzle is by the row modulo 8; codes past the end of a row: zeros
        auto rows = [&](uint32_t dst, const uint8_t *tile, int last, uint32_t byte) {
            const bool in = byte + seg < pitch;
            const uint8_t *src = tile + (in ? byte : 0);
            const int r0 = cw * kInstr * 4 + (lane >> 3);
#pragma unroll
            for (int j = 0; j < kInstr; ++j) {
                const int r = r0 + j * 4;
                copy_async_16(dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4), src + (size_t)(uint32_t)(r < last ? r : last) * pitch, in);
            }
        };
        // (rows past the last one are read from it again: nothing of them is stored)
        auto begin = [&](int tile) {
            const int n0 = tile / m_tiles * C::kChannels, m0 = tile % m_tiles * kPairTok + (int)rank * kPairHalf;
            const int nr = n0 + (GATED ? 0 : (int)rank * 128), nb = nr < N ? nr : N - 1, mb = m0 < M ? m0 : M - 1;
            wtile = wrows + (size_t)nb * pitch + seg, w_last = N - 1 - nb;
            xtile = x_codes + (size_t)mb * pitch + seg, x_last = M - 1 - mb;
#pragma unroll
            for (int j = 0; j < C::kPieces / 2; ++j) {
                const int c = j * 128 + t, half = c / (C::kPieces * 32), nt = (n0 >> 7) + (GATED ? 0 : half);
                sfw_src[j] = (GATED && half ? w2_pieces : w_pieces) + (size_t)(nt < last_n ? nt : last_n) * pieces * 512 + (c % (C::kPieces * 32)) * 16;
            }
            sfx_src = x_pieces + (size_t)((m0 >> 7) < last_m ? m0 >> 7 : last_m) * pieces * 512 + t * 16;
        };
        auto copy_w = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t sf = (size_t)i * C::kPieces * 512;
            rows(dst + C::kBOff, wtile, w_last, (uint32_t)i * kFp4RowBytes);
#pragma unroll
            for (int j = 0; j < C::kPieces / 2; ++j) copy_async_16(dst + C::kSfbOff + (j * 128 + t) * 16, sfw_src[j] + sf, true);
        };
        auto copy_x = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t sf = (size_t)i * C::kPieces * 512;
            rows(dst, xtile, x_last, (uint32_t)i * kFp4RowBytes);
            if (t < C::kSfaBytes / 16) copy_async_16(dst + C::kSfaOff + t * 16, sfx_src + sf, true);
        };
        begin(pair);
        const int pre = rounds < C::kStages ? rounds : C::kStages;
        for (int i = group; i < pre; i += 2) copy_w(i, i);
        pdl_wait();
        int it = 0;  // stages so far, of both groups
        uint32_t s = 0, ph = 0;
        auto bring = [&](int first, int last) {
            for (int i = first; i < last; ++i, ++it) {
                if ((it & 1) == group) {
                    if (it >= C::kStages) mbar_wait_lane<kTimeoutFp4Pair, 0>(bars + kEmptyBar + s * 8, ph ^ 1u, ctl, status, 0, s);
                    if (it >= pre) copy_w(i, s);
                    copy_x(i, s);
                    copy_async_arrive(bars + kFullBar + s * 8);
                }
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        };
        // the next tile's first stages are requested before this tile is finished
        bring(0, pre);
        for (int tile = pair; tile < tiles; tile += pairs) {
            bring(pre, rounds);
            if (tile + pairs < tiles) {
                begin(tile + pairs);
                bring(0, pre);
            }
            finish(tile);
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
