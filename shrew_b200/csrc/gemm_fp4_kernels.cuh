// Forward of a layer whose weights and activations are both 4-bit microscaled codes, on the block-scaled tensor cores (tcgen05.mma
// kind::mxf4 and kind::mxf4nvf4), sm_100a only.
//
//   y[m,n] = epi( alpha[n] * sum_k (w code * w scale)[n,k] (x code * x scale)[m,k] + bias[n] ),  f32 sums
//
// Mapping.  D[128 x TOK] += A[128 x 64] * B[TOK x 64]^T for each instruction: A = 128 weight rows, B = a tile of tokens, both packed codes in
// shared memory (128-byte swizzle, K-major: one row of a stage is 256 codes = 128 bytes), D = f32 accumulators in tensor memory
// (lane = output channel, column = token).  The scales of a stage are the 512-byte pieces that the quantizer and the handle lay out
// (scale_piece_offset); they go on to tensor memory with tcgen05.cp just ahead of the MMAs that use them, every stage of the ring into
// columns of its own, so that the release of the stage covers them too.
//
// What bounds a wide tile is getting 51 KB a stage into the SM: at the matrix rate a stage lasts 512 cycles.  TMA moves a row of a box in
// some 4 cycles whatever its length (measured: 16 / 29 / 47 bytes a cycle and SM with rows of 64 / 128 / 256 bytes, and the swizzle allows
// 128), cp.async 64 to 67; 384 rows by TMA were 1470 cycles.  So the eight epilogue warps, idle until the end, bring the stages with cp.async,
// 16 bytes a lane, swizzled as they land.  The copies arrive on the stage's barrier by themselves, a relay warp makes them visible to the
// tensor core, and the thread that issues the MMAs looks for the next stage while it issues this one's: 4096 x 4096 with 32 tokens 9.3 -> 8.8 us
// (8.0 with TMA, which is quicker to start and slower from 64 tokens on; batches that fill the machine go to gemm_fp4_pair_kernels.cuh).
//
// GATED: two MMAs into two accumulators: gate rows and up rows of the same 128 channels against the same token tile; a lane then
// holds both values of its channel and the epilogue writes silu(gate) * up without an exchange.
//
// The k range of a tile may be split over a cluster (tcgen05_cluster_epilogue.cuh).
//
// Warp roles: warp 0 = tensor-memory allocation and MMA issue, then 8 warps that copy and, at the end, run the epilogue, then the relay.
// full[s] (the copies of 256 threads) -> relay -> ready[s] -> MMA -> empty[s] (tcgen05.commit) -> copies; every wait is bounded as in the
// other tcgen05 kernels.
// Programmatic dependent launch: weights of the first stages are requested before the wait for the previous kernel, the activations'
// codes (the quantizer's output) after it.
//
// Device code only; also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "../../include/shrewq.h"
#include "dests.cuh"
#include "ptx_fp4.cuh"
#include "ptx_small.cuh"
#include "ptx_tcgen05.cuh"
#include "ptx_tcgen05_fp4.cuh"
#include "tcgen05_cluster_epilogue.cuh"
#include "tcgen05_common.cuh"

namespace shrewq {
namespace {

constexpr int kFp4StageK = 256;       // codes of k a stage: rows of 128 bytes
constexpr int kFp4RowBytes = 128;
constexpr int kFp4Groups = 2;         // groups of 4 warps that copy and run the epilogue
constexpr int kFp4Copiers = 4 * kFp4Groups, kFp4GemmThreads = 32 + 32 * kFp4Copiers + 32;
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
    static constexpr int kSlotOff = kFp4Groups * kEpiStageBytes;           // received sums behind the staging tiles
    static_assert(kStages * kStageBytes >= kSlotOff + ClusterEpi<TOK, GATED ? kEpiColumns : kEpiPlain>::kSlotBytes, "the epilogue reuses the stages");
};

__device__ __forceinline__ bool fp4_wait(uint32_t bar, uint32_t parity, Ctl *ctl, DeviceStatus *st, uint32_t role, uint32_t stage) {
    return mbar_wait_close<kTimeoutFp4>(bar, parity, ctl, st, role, stage);
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

// `rows` rows of 128 bytes of a K-major operand into a swizzled tile: 4 rows an instruction, the warp's share of them.  src: the lane's first
// row and 16-byte piece; rows past `last` repeat it (what they give is not stored).
template <int ROWS>
struct CopyRows {
    static constexpr int kInstr = ROWS / 4 / kFp4Copiers;  // of a warp
    const uint8_t *src[kInstr];
    __device__ __forceinline__ CopyRows(const uint8_t *base, size_t pitch, int row0, int last, int copier, int lane) {
#pragma unroll
        for (int j = 0; j < kInstr; ++j) {
            const int r = row0 + (copier * kInstr + j) * 4 + (lane >> 3);
            src[j] = base + (size_t)(r < last ? r : last) * pitch + (lane & 7) * 16;
        }
    }
    // `in`: false = zeros
    __device__ __forceinline__ void copy(uint32_t tile, size_t byte, int copier, int lane, bool in) const {
#pragma unroll
        for (int j = 0; j < kInstr; ++j) {
            const int r = (copier * kInstr + j) * 4 + (lane >> 3);
            copy_async_16(tile + r * 128 + (((lane & 7) ^ (r & 7)) << 4), in ? src[j] + byte : src[j], in);
        }
    }
};

template <int TOK, bool NV, bool GATED, typename YT>
__global__ void __launch_bounds__(kFp4GemmThreads, 1)
gemm_fp4_kernel(const uint8_t *__restrict__ w_codes, const uint8_t *__restrict__ w2_codes, const uint8_t *x_codes, const uint8_t *__restrict__ w_pieces,
                const uint8_t *__restrict__ w2_pieces, const uint8_t *x_pieces, Operands ops, YT *__restrict__ y, int M, int N, int K, size_t ldy,
                int epilogue, int S, int rounds_per_cta, DeviceStatus *status) {
    using C = Fp4Cfg<TOK, NV, GATED>;
    pdl_launch_dependents();
    SHREWQ_DYNAMIC_SMEM(uint8_t, smem_raw);
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bar_area = smem + C::kStages * C::kStageBytes;
    Ctl *ctl = reinterpret_cast<Ctl *>(bar_area + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // token tiles fastest: the CTAs that share a weight tile start together, so it comes from DRAM once
    const int m_tiles = (M + TOK - 1) / TOK;
    constexpr int kMode = GATED ? kEpiColumns : kEpiPlain;
    // (the rank from the block's index: a value that the compiler knows to be the same in all lanes, as the operands of tcgen05
    // instructions are that derive from it)
    const uint32_t rank = blockIdx.x % (unsigned)S;
    const int tile = (int)(blockIdx.x / (unsigned)S);
    const int m0 = tile % m_tiles * TOK, n0 = tile / m_tiles * 128;
    const int rounds_total = (K + kFp4StageK - 1) / kFp4StageK, r_begin = (int)rank * rounds_per_cta;
    const int rounds = min(rounds_total - r_begin, rounds_per_cta);  // >= 1 by construction of the grid
    const size_t pieces = (size_t)rounds_total * C::kPieces;  // along a row
    constexpr uint32_t kFullBar = 0, kEmptyBar = C::kStages * 8, kReadyBar = 2 * C::kStages * 8, kAccBar = 3 * C::kStages * 8;
    const uint32_t bars = smem_u32(bar_area), smem_base = smem_u32(smem);

    if (threadIdx.x == 0) {
        ctl->abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bars + kFullBar + s * 8, 32 * kFp4Copiers);
            mbar_init(bars + kReadyBar + s * 8, 1);
            mbar_init(bars + kEmptyBar + s * 8, 1);
        }
        mbar_init(bars + kAccBar, 1);
        mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        tc_alloc_512(smem_u32(&ctl->tmem_base));
        tc_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, ctl->tmem_base, 0);  // (uniform to the compiler)
    bool ok = true;
    const int copier = warp - 1, group = copier >> 2, quad = warp & 3;
    const bool epi = warp >= 1 && warp <= kFp4Copiers;

    if (warp == 0) {
        if (elect_one()) {
            pdl_wait();  // a stage is full only with its activations: the time limit of the waits starts when they exist
            uint32_t s = 0, ph = 0;
            bool good = true, ready = false;
            for (int i = 0; i < rounds; ++i) {
                good = ready || fp4_wait(bars + kReadyBar + s * 8, ph, ctl, status, 1, s);
                if (!good) break;
                tc_fence_after();
                // (a look takes 150 to 300 cycles here: the next stage's is under way while this one's MMAs are issued)
                const uint32_t next = s + 1 == C::kStages ? 0 : s + 1, next_ph = s + 1 == C::kStages ? ph ^ 1u : ph;
                ready = mbar_test(bars + kReadyBar + next * 8, next_ph);
                const uint32_t base = smem_base + s * C::kStageBytes;
                const uint32_t sf = tmem + C::kAccCols + s * C::kSfCols;             // A pieces (gate, up), then B pieces
                constexpr int kSfbCol = C::kMats * C::kPieces * 4, kBStep = 4 * C::kTokTiles;
                // descriptors of this stage: every other one is a constant away (16-byte units; the address field does not overflow)
                const uint64_t adesc = make_b_desc(base), bdesc = make_b_desc(base + C::kBOff), sdesc = make_scale_desc(base + C::kSfaOff);
                const uint32_t tok_col = TOK < 128 ? (uint32_t)((m0 & 127) >> 5) : 0u;  // a token tile of half a piece
#pragma unroll
                for (int p = 0; p < C::kPieces; ++p) {
                    const uint32_t sfa = sf + p * 4, sfb = sf + kSfbCol + p * kBStep;
#pragma unroll
                    for (int a = 0; a < C::kMats; ++a) tc_cp_scales(sfa + a * C::kPieces * 4, sdesc + (uint64_t)((a * C::kPieces + p) * 32));
#pragma unroll
                    for (int j = 0; j < C::kTokTiles; ++j)
                        tc_cp_scales(sfb + j * 4, sdesc + (uint64_t)(((C::kSfbOff - C::kSfaOff) >> 4) + (j * C::kPieces + p) * 32));
                    // a piece covers 64 codes (NV) or 128 (MX: two MMAs, the second with the upper half of the scale bytes)
#pragma unroll
                    for (int h = 0; h < 4 / C::kPieces; ++h) {
                        const int q = p * (4 / C::kPieces) + h;  // 64 codes = 32 bytes of a row
#pragma unroll
                        for (int a = 0; a < C::kMats; ++a)
                            tc_mma_fp4<NV>(tmem + a * TOK, adesc + (uint64_t)((a * C::kABytes + q * 32) >> 4), bdesc + (uint64_t)((q * 32) >> 4),
                                           fp4_idesc(NV, 128, TOK, (uint32_t)h * 2u), sfa + a * C::kPieces * 4, sfb + tok_col, (i > 0 || q > 0) ? 1u : 0u);
                    }
                }
                tc_commit(bars + kEmptyBar + s * 8);
                s = next, ph = next_ph;
            }
            if (good) tc_commit(bars + kAccBar);
        }
        __syncwarp();
    } else if (warp == kFp4GemmThreads / 32 - 1) {
        // ---------------- relay: copies that have landed -> visible to the tensor core -> the MMAs ----------------
        if (elect_one()) {
            pdl_wait();
            uint32_t s = 0, ph = 0;
            for (int i = 0; i < rounds; ++i) {
                if (!fp4_wait(bars + kFullBar + s * 8, ph, ctl, status, 5, s)) break;
                fence_proxy_async_smem();
                mbar_arrive(bars + kReadyBar + s * 8);
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else {
        // ---------------- copies, then the epilogue ----------------
        const size_t pitch = (size_t)((K + 31) >> 5) * 16;
        const int t = (int)threadIdx.x - 32;  // 0 .. 255
        const CopyRows<128> gate_rows(w_codes, pitch, n0, N - 1, copier, lane), up_rows(w2_codes, pitch, n0, N - 1, copier, lane);
        const CopyRows<TOK> token_rows(x_codes, pitch, m0, M - 1, copier, lane);
        auto copy_w = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t byte = (size_t)(r_begin + i) * kFp4RowBytes;
            const bool in = byte + (lane & 7) * 16 < pitch;  // (codes past the end of a row: zeros)
            gate_rows.copy(dst, byte, copier, lane, in);
            if constexpr (GATED) up_rows.copy(dst + C::kABytes, byte, copier, lane, in);
            const size_t at = ((size_t)(n0 >> 7) * pieces + (size_t)(r_begin + i) * C::kPieces) * 512;
            if (t < C::kMats * C::kSfaBytes / 16) {
                const int mat = GATED ? t / (C::kSfaBytes / 16) : 0, c = t % (C::kSfaBytes / 16);
                copy_async_16(dst + C::kSfaOff + t * 16, (mat ? w2_pieces : w_pieces) + at + c * 16, true);
            }
        };
        // the token tiles of the pieces beyond the last one are read from it again: their columns are not stored
        const int last_tile = (M - 1) >> 7;
        auto copy_x = [&](int i, int s) {
            const uint32_t dst = smem_base + s * C::kStageBytes;
            const size_t byte = (size_t)(r_begin + i) * kFp4RowBytes;
            token_rows.copy(dst + C::kBOff, byte, copier, lane, byte + (lane & 7) * 16 < pitch);
            if (t < C::kSfbBytes / 16) {
                const int j = t / (C::kPieces * 32), c = t % (C::kPieces * 32);
                const int xt = (m0 >> 7) + j < last_tile ? (m0 >> 7) + j : last_tile;
                copy_async_16(dst + C::kSfbOff + t * 16, x_pieces + ((size_t)xt * pieces + (size_t)(r_begin + i) * C::kPieces) * 512 + c * 16, true);
            }
        };
        const int pre = rounds < C::kStages ? rounds : C::kStages;
        for (int i = 0; i < pre; ++i) copy_w(i, i);
        pdl_wait();  // (and y may be in use by the previous kernel of the stream)
        for (int i = 0; i < rounds; ++i) {
            const int s = i % C::kStages;
            if (i >= C::kStages) {
                mbar_wait_all<kTimeoutFp4>(bars + kEmptyBar + s * 8, (uint32_t)(i / C::kStages - 1) & 1u, ctl, status, 0, s);
                copy_w(i, s);
            }
            copy_x(i, s);
            copy_async_arrive(bars + kFullBar + s * 8);
        }
        mbar_wait_all<kTimeoutFp4>(bars + kAccBar, 0, ctl, status, 4, 0);
        ok = warp_ok(ctl);
        tc_fence_after();
        if (S == 1)
            cluster_finish<TOK, kFp4Groups, kMode, YT>(tmem, smem, nullptr, 1, 0, group, quad, lane, ok, ops, y, M, N, ldy, epilogue, n0, m0);
    }
    if (S > 1) {
        tc_fence_before();
        __syncwarp();
        cluster_arrive();  // every CTA of the tile has its sums: the stages are idle everywhere
        cluster_wait();
        tc_fence_after();
        if (epi && ok) cluster_send<TOK, kFp4Groups, kMode>(tmem, smem_base + C::kSlotOff, S, rank, group, quad, lane);
        __syncwarp();
        cluster_arrive();  // and has received the others'
        cluster_wait();
        if (epi)
            cluster_finish<TOK, kFp4Groups, kMode, YT>(tmem, smem, reinterpret_cast<const float *>(smem + C::kSlotOff), S, rank, group, quad, lane, ok, ops, y, M, N,
                                                       ldy, epilogue, n0, m0);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (ctl->abort_flag) {
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // MMAs in flight get a bounded moment to land
        }
        tc_fence_after();
        __syncwarp();
        tc_dealloc_512(tmem);
    }
}

}  // namespace
}  // namespace shrewq
