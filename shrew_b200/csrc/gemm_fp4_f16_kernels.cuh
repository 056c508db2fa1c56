// Forward of a layer with 4-bit microscaled weights for up to 32 tokens, on the tensor cores (tcgen05.mma kind::f16 in f16), sm_100a only.
// (linear_fp4.cu says which calls take it: in the main 5 to 32 bf16 tokens over more tiles than SMs.)
//
//   y[m,n] = epi( alpha[n] * 2^e[m] * sum_k w[n,k] x'[m,k] + bias[n] ),   x' = x * 2^-e[m] in f16 terms
//
// Bound by the weight stream (0.53 or 0.56 bytes a weight).  mma.sync is no way to keep up with it here: an m16n8k16 holds its tensor pipe
// for 32 cycles (measured: 75 % busy at 16 tokens with the stream at a fifth of its rate), where one tcgen05.mma multiplies
// 128 rows by the tokens.  So the weights go the way of the large forward, widened by converter warps into TENSOR MEMORY, but in f16:
// one conversion for two codes and one packed multiplication by the block scale, 1 issue slot a code against 2.5 in bf16.  What f16 cannot
// hold at once takes further passes over the codes, as in gemv_fp4_kernels.cuh: windows of 28 octaves of MX scales, and f16 terms of the
// activations where a token has values below 2^-32 of its largest (f32: three terms of 11 bits).  Each pass's sums are added in f32 with
// their power of two to totals in tensor memory; with one pass (all ordinary tensors) nothing of that runs, and the rounds' products go to four
// accumulators in turn (two for more than 16 tokens), added in f32 at the end: a chain into one loses what is below its last place at every step.
// Gated 11008 x 4096 NV with 8 and 16 tokens: sums 5.2e-7 -> 1.2e-7 off, bf16 results 9e-5 -> 1.3e-5 from those of exact sums, 24.4 -> 24.8 us.
//
// Two CTAs share an SM (256 columns of tensor memory, half the shared memory): up to 296 tiles are in flight at once, and one CTA's prologue and
// epilogue hide behind the other's loads.  What an SM takes in bounds it, some 16 bytes a cycle for the 64-byte rows of its boxes, so the time is that
// of the SMs with two tiles: 172 gated tiles (11008 x 4096, 16 tokens) 26 us, 296 tiles 27.7, 148 tiles 21.1, from cold HBM, staging included.
// Mapping otherwise as gemm_fp4_bf16_kernels.cuh: D[128 x TOK] += A[128 x 16] B[TOK x 16]^T, stages of 128 codes a row, GATED tiles
// interleave 64 gate and 64 up rows, k split over a cluster.  Codes and activations wait in a ring of kStages in shared memory; the
// widened codes have kSlots places in tensor memory.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "../../include/shrewq.h"
#include "fp4_kernels.cuh"
#include "fp4_params.cuh"
#include "gemv_fp4_kernels.cuh"
#include "ptx_small.cuh"
#include "ptx_tcgen05.cuh"
#include "ptx_tcgen05_fp4.cuh"
#include "tcgen05_cluster_epilogue.cuh"
#include "tcgen05_common.cuh"

namespace shrewq {
namespace {

constexpr int kH4StageK = 128, kH4Groups = 3, kH4Threads = 64 + 128 * kH4Groups;
constexpr uint32_t kTimeoutH4 = 7;  // DeviceStatus::timeout_flag of this kernel

template <int TOK, bool NV, bool GATED>
struct H4Cfg {
    static constexpr int kCodeBytes = 128 * (kH4StageK / 2);
    static constexpr int kXBox = TOK * 128, kXBytes = 2 * kXBox;          // 64 f16 of every token, twice
    static constexpr int kMats = GATED ? 2 : 1, kPieces = NV ? 2 : 1;
    static constexpr int kScaleBytes = kMats * kPieces * 512;
    static constexpr int kXOff = kCodeBytes, kScaleOff = kXOff + kXBytes;
    static constexpr int kTxBytes = kCodeBytes + kXBytes + kScaleBytes;
    static constexpr int kStageBytes = (kTxBytes + 1023) / 1024 * 1024;
    static constexpr int kStages = 6, kSlots = kH4Groups;                  // (kStages a multiple of the groups, see the converters)
    static constexpr int kACols = kH4StageK / 2, kABase = 64;              // tensor memory: sums (one pass) or sums and totals (several), widened codes
    static constexpr int kAccs = kABase / TOK;                             // accumulators of a single pass
    static constexpr int kSmemBytes = kStages * kStageBytes + 2048;
    static constexpr int kSlotOff = 2 * kEpiStageBytes;                    // (at most two chunks of 16 tokens: two groups have staging tiles)
    static_assert(kABase >= 2 * TOK && (kAccs & (kAccs - 1)) == 0 && kABase + kSlots * kACols <= 256 && kStages % kH4Groups == 0, "tensor memory of half an SM");
    // What is asked for is half an SM's shared memory, and enough that a kernel which takes all of tensor memory (they ask for 120 KB) never
    // shares an SM with this one: of two such neighbours in a stream, started early, one could hold the memory that the other waits for.
    static constexpr int kSmemRequest = 110 * 1024;
    static_assert(kSmemBytes <= kSmemRequest && 2 * (kSmemRequest + 1024) <= 228 * 1024 && kSmemRequest + 1024 + 121 * 1024 > 228 * 1024, "shared memory");
    static_assert(kStages * kStageBytes >= kSlotOff + ClusterEpi<TOK, kEpiPlain>::kSlotBytes, "the epilogue reuses the stages");
};

// 32 codes (16 bytes) and their factors -> 16 packed f16x2, natural order
__device__ __forceinline__ void widen32_f16(const uint4 c, uint32_t f_lo, uint32_t f_hi, uint32_t *out) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        cvt_f16x8_e2m1(w[q], out + 4 * q);
#pragma unroll
        for (int p = 0; p < 4; ++p) out[4 * q + p] = mul_f16x2(out[4 * q + p], q < 2 ? f_lo : f_hi);
    }
}

// x: terms of M rows, `most` of them stacked (tmap_x); exps, counts: by token
template <int TOK, bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kH4Threads, 2)
gemm_w4_f16_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w2, const __grid_constant__ CUtensorMap tmap_x, Fp4Operand w0,
                   Fp4Operand w1, const float *__restrict__ alpha0, const float *__restrict__ alpha1, const int *exps, const int *counts,
                   int most, int octaves, YT *__restrict__ y, int M, int N, int K, size_t ldy, int epilogue, int S, int rounds_per_cta, DeviceStatus *status) {
    using C = H4Cfg<TOK, NV, GATED>;
    constexpr int kChan = GATED ? 64 : 128, kMode = GATED ? kEpiLanesPaired : kEpiPlain;
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem_raw);
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bar_area = smem + C::kStages * C::kStageBytes;
    Ctl *ctl = reinterpret_cast<Ctl *>(bar_area + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % (unsigned)S;
    const int n0 = (int)(blockIdx.x / (unsigned)S) * kChan;   // (one token tile: M <= TOK)
    const int rounds_total = (K + kH4StageK - 1) / kH4StageK, r_begin = (int)rank * rounds_per_cta;
    const int rounds = min(rounds_total - r_begin, rounds_per_cta);  // of a pass; >= 1 by construction of the grid
    const size_t pieces = (size_t)((K + 255) >> 8) * (NV ? 4 : 2);
    constexpr uint32_t kFullBar = 0, kEmptyBar = C::kStages * 8, kAreadyBar = 2 * C::kStages * 8, kAfreeBar = kAreadyBar + C::kSlots * 8,
                       kAccBar = kAfreeBar + C::kSlots * 8, kTakenBar = kAccBar + 8;
    const uint32_t bars = smem_u32(bar_area), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 1);
            mbar_init(bars + kEmptyBar + s * 8, 1);
        }
        for (int s = 0; s < C::kSlots; ++s) {
            mbar_init(bars + kAreadyBar + s * 8, 4);
            mbar_init(bars + kAfreeBar + s * 8, 1);
        }
        mbar_init(bars + kAccBar, 1);
        mbar_init(bars + kTakenBar, 4 * kH4Groups);
        mbar_fence_init();
    }
    if (warp == 1) {
        tc_alloc_256(smem_u32(&ctl->tmem_base));  // (column 256 for the second CTA of an SM; nobody else writes the word)
        tc_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, ctl->tmem_base, 0);  // (uniform to the compiler)
    // the next kernel of the stream may start, now that this one has its tensor memory: it will wait for this one to end, with whatever it
    // has allocated on this SM
    pdl_launch_dependents();
    bool ok = true;

    auto load_w = [&](int r, int s) {  // round r of this CTA's part of k into stage s
        const uint32_t dst = smem_base + s * C::kStageBytes, fb = bars + kFullBar + s * 8;
        mbar_expect_tx(fb, C::kTxBytes);
        const size_t at = ((size_t)(n0 >> 7) * pieces + (size_t)(r_begin + r) * C::kPieces) * 512;
        tma_load_2d(dst, &tmap_w, (r_begin + r) * (kH4StageK / 2), n0, fb);
        bulk_load_1d(dst + C::kScaleOff, w0.pieces + at, C::kPieces * 512, fb);
        if constexpr (GATED) {
            tma_load_2d(dst + 64 * (kH4StageK / 2), &tmap_w2, (r_begin + r) * (kH4StageK / 2), n0, fb);
            bulk_load_1d(dst + C::kScaleOff + C::kPieces * 512, w1.pieces + at, C::kPieces * 512, fb);
        }
    };
    auto load_x = [&](int r, int term, int s) {
        const uint32_t dst = smem_base + s * C::kStageBytes + C::kXOff, fb = bars + kFullBar + s * 8;
        tma_load_2d(dst, &tmap_x, (r_begin + r) * kH4StageK, term * M, fb);
        tma_load_2d(dst + C::kXBox, &tmap_x, (r_begin + r) * kH4StageK + 64, term * M, fb);
    };
    const int pre = rounds < C::kStages ? rounds : C::kStages;  // stages of the first pass that are free at the start
    if (warp == 0 && elect_one())
        for (int i = 0; i < pre; ++i) load_w(i, i);
    __syncwarp();
    pdl_wait();  // activations are the staging kernel's; y may be in use before

    // passes: the terms that any token needs times the windows of the scales
    int n_terms = 1;
    for (int m = lane; m < M; m += 32) n_terms = ld_written_s32(counts + m);
    n_terms = (int)warp_max((unsigned int)n_terms);
    n_terms = n_terms < most ? n_terms : most;
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
    const int passes = n_terms * windows, items = passes * rounds;
    // accumulators in turn (uniform to the compiler: an operand of the matrix instructions derives from it), and those that hold something
    const int accs = __shfl_sync(0xFFFFFFFFu, passes == 1 ? C::kAccs : 1, 0), parts = rounds < accs ? rounds : accs;

    if (warp == 0) {
        if (elect_one()) {
            for (int i = 0; i < pre; ++i) load_x(i, 0, i);
            uint32_t s = pre == C::kStages ? 0 : (uint32_t)pre, ph = pre == C::kStages ? 0u : 1u;
            int pass = pre == rounds ? 1 : 0, r = pre == rounds ? 0 : pre;
            for (int i = pre; i < items; ++i) {
                // a stage of the first round through the ring is free: the wait for the phase before it returns at once
                if (!mbar_wait_close<kTimeoutH4>(bars + kEmptyBar + s * 8, ph, ctl, status, 0, s)) break;
                load_w(r, (int)s);
                load_x(r, pass / windows, (int)s);
                if (++s == C::kStages) { s = 0; ph ^= 1; }
                if (++r == rounds) { r = 0; ++pass; }
            }
        }
    } else if (warp == 1) {
        // D=f32, A=f16 (tensor memory), B=f16 (K-major), M=128, N=TOK
        constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(TOK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        uint32_t s = 0, slot = 0, slot_ph = 0;
        bool good = true;
        if (elect_one()) {
            for (int pass = 0; pass < passes && good; ++pass) {
                // the sums of the pass before have been taken out, and every converter warp has seen them complete
                if (pass > 0) good = mbar_wait_close<kTimeoutH4>(bars + kTakenBar, (uint32_t)(pass - 1) & 1u, ctl, status, 5, 0);
                for (int i = 0; i < rounds && good; ++i) {
                    // (the converters have waited for the stage: its activations are there too)
                    good = mbar_wait_close<kTimeoutH4>(bars + kAreadyBar + slot * 8, slot_ph, ctl, status, 2, slot);
                    if (!good) break;
                    tc_fence_after();
                    const uint64_t bdesc = make_b_desc(smem_base + s * C::kStageBytes + C::kXOff);
                    const uint32_t a = tmem + C::kABase + slot * C::kACols, d = tmem + (uint32_t)(i & (accs - 1)) * TOK;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            tc_mma_ts_f16(d, a + j * 32 + q * 8, bdesc + (uint64_t)((j * C::kXBox + q * 32) >> 4), idesc, (i >= accs || j > 0 || q > 0) ? 1u : 0u);
                    tc_commit(bars + kAfreeBar + slot * 8);  // frees the place of its widened codes ...
                    tc_commit(bars + kEmptyBar + s * 8);     // ... and the stage
                    if (++s == C::kStages) s = 0;
                    if (++slot == C::kSlots) { slot = 0; slot_ph ^= 1; }
                }
                if (good) tc_commit(bars + kAccBar);
            }
        }
        __syncwarp();
    } else {
        const int group = (warp - 2) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const int srow = GATED ? (row & 1) * 64 + (row >> 1) : row, swz = (srow >> 1) & 3;
        const int prow = GATED ? (n0 & 64) + (row >> 1) : row;
        const int scale_at = C::kScaleOff + (GATED ? (row & 1) * C::kPieces * 512 : 0) + (prow & 31) * 16 + (prow >> 5) * 4;
        int item = 0;
        for (int pass = 0; pass < passes; ++pass) {
            const int first = top - (kMxWindow - 1) - kMxWindow * (pass % windows);  // MX: the byte of 2^-14 in this window
            for (int i = 0; i < rounds; ++i, ++item) {
                // group g takes the items i % 3 == g, and so, the ring being a multiple, always the same stages and place: it passes through
                // every phase of their barriers, so that a wait for a parity cannot take one phase for another
                const int slot = item % C::kSlots, s = item % C::kStages;
                if (slot != group) continue;
                mbar_wait_all<kTimeoutH4>(bars + kFullBar + s * 8, (uint32_t)(item / C::kStages) & 1u, ctl, status, 3, s);
                const uint8_t *stage = smem + s * C::kStageBytes;
                uint32_t scales[2];
                scales[0] = *reinterpret_cast<const uint32_t *>(stage + scale_at);
                if constexpr (NV) scales[1] = *reinterpret_cast<const uint32_t *>(stage + scale_at + 512);
#pragma unroll
                for (int b = 0; b < 4; ++b) {  // 32 codes
                    uint32_t f0, f1, packed[16];
                    if constexpr (NV) {
                        const uint32_t two = cvt_f16x2_e4m3(scales[b >> 1] >> (16 * (b & 1)));
                        f0 = dup_lo(two);
                        f1 = dup_hi(two);
                    } else {
                        f0 = f1 = mx_scale_f16x2(scales[0], b, first);
                    }
                    widen32_f16(*reinterpret_cast<const uint4 *>(stage + srow * (kH4StageK / 2) + ((b ^ swz) << 4)), f0, f1, packed);
                    if (b == 0) {  // the MMAs of this group's item before have read their codes
                        if (item >= C::kSlots)
                            mbar_wait_all<kTimeoutH4>(bars + kAfreeBar + slot * 8, (uint32_t)(item / C::kSlots - 1) & 1u, ctl, status, 6, slot);
                        tc_fence_after();
                    }
                    tc_st16(tmem + lanes + C::kABase + slot * C::kACols + b * 16, packed);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bars + kAreadyBar + slot * 8);
            }
            mbar_wait_all<kTimeoutH4>(bars + kAccBar, (uint32_t)pass & 1u, ctl, status, 4, 0);
            ok = warp_ok(ctl);
            tc_fence_after();
            if (passes > 1) {
                // the first group adds the pass's sums to the totals, which take the sums' place in the end
                if (group == 0) {
                    const float weight = ldexpf(1.0f, -octaves * (pass / windows) - kMxWindow * (pass % windows));
                    const bool last = pass + 1 == passes;
#pragma unroll 1
                    for (int c = 0; c < TOK; c += 16) {
                        uint32_t r[16], t[16];
                        tc_ld16(tmem + lanes + c, r);
                        tc_ld16(tmem + lanes + TOK + c, t);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            t[i] = __float_as_uint(pass == 0 ? __uint_as_float(r[i]) : __fmaf_rn(__uint_as_float(r[i]), weight, __uint_as_float(t[i])));
                        tc_st16(tmem + lanes + (last ? 0 : TOK) + c, t);
                    }
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                }
                // Every warp, so that none can miss a phase of the accumulators' barrier: a group without an item in some passes (a round or
                // two of them) would otherwise be held back by nothing, and two phases later its parity reads as if none had been.
                if (lane == 0 && pass + 1 < passes) mbar_arrive(bars + kTakenBar);
                if (pass + 1 == passes) {
                    named_bar_sync(1, 128 * kH4Groups);
                    tc_fence_after();
                }
            }
        }
        if (S == 1)
            cluster_finish<TOK, kH4Groups, kMode, YT, true>(tmem, smem, nullptr, 1, 0, group, quad, lane, ok, Operands{alpha0, w0.bias, alpha1, w1.bias}, y, M, N, ldy,
                                                            epilogue, n0, 0, exps, NV ? 0 : top - 140, parts);
    }
    if (S > 1) {
        const int group = (warp - 2) >> 2, quad = warp & 3;
        tc_fence_before();
        __syncwarp();
        cluster_arrive();  // every CTA of the tile has its sums: the stages are idle everywhere
        cluster_wait();
        tc_fence_after();
        if (warp >= 2 && ok) cluster_send<TOK, kH4Groups, kMode>(tmem, smem_base + C::kSlotOff, S, rank, group, quad, lane, parts);
        __syncwarp();
        cluster_arrive();  // and has received the others'
        cluster_wait();
        if (warp >= 2)
            cluster_finish<TOK, kH4Groups, kMode, YT, true>(tmem, smem, reinterpret_cast<const float *>(smem + C::kSlotOff), S, rank, group, quad, lane, ok,
                                                            Operands{alpha0, w0.bias, alpha1, w1.bias}, y, M, N, ldy, epilogue, n0, 0, exps, NV ? 0 : top - 140, parts);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (ctl->abort_flag) {
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies and MMAs in flight get a bounded moment to land
        }
        tc_fence_after();
        __syncwarp();
        tc_dealloc_256(tmem);
    }
}

}  // namespace
}  // namespace shrewq
