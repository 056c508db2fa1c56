// Stand-ins for shrew_b200/csrc/ptx_tcgen05_fp4.cuh: tcgen05.cp of block scales and the block-scaled tcgen05.mma on E2M1 operands.
// Include after cuda_shim_tcgen05.h and cuda_shim_fp4.h.  TEST INFRASTRUCTURE ONLY.
#pragma once

namespace emu {
inline uint32_t desc_start(uint64_t d) { return (uint32_t)(d & 0x3FFFu) << 4; }
inline uint32_t desc_stride(uint64_t d) { return (uint32_t)((d >> 32) & 0x3FFFu) << 4; }
inline float scale_value(bool nv, uint32_t byte) { return nv ? emu_e4m3_value(byte & 0x7F) : byte == 255 ? NAN : ldexpf(1.0f, (int)byte - 127); }
// E2M1 value (row, k) of a K-major operand with 128-byte swizzle; rows of 128 bytes, 8-row groups `stride` apart
inline float fp4_operand(Block *blk, uint64_t desc, uint32_t row, uint32_t k) {
    const uint32_t addr = (smem_u32(blk->dyn) | desc_start(desc)) + (row >> 3) * desc_stride(desc) + (row & 7) * 128 + (k >> 1);
    const uint8_t byte = *smem_ptr(swizzle(addr, 128));
    return emu_e2m1_value(k & 1 ? byte >> 4 : byte & 15);
}
inline void cp_scales(Block *blk, uint32_t taddr, uint64_t desc) {
    const uint32_t col = taddr & 0xFFFF;
    if ((taddr >> 16) != 0 || col + 4 > 512) { fail("tcgen05.cp outside tensor memory"); return; }
    EMU_CHECK(((desc >> 61) & 7u) == 0 && ((desc >> 46) & 1u) == 1, "scales: no swizzle, descriptor version 1");
    for (uint32_t r = 0; r < 32; ++r) {
        const uint8_t *src = smem_ptr((smem_u32(blk->dyn) | desc_start(desc)) + (r >> 3) * desc_stride(desc) + (r & 7) * 16);
        for (uint32_t j = 0; j < 4; ++j) {
            uint32_t w;
            memcpy(&w, src + 4 * j, 4);
            for (uint32_t q = 0; q < 4; ++q) blk->tmem[(q * 32 + r) * 512 + col + j] = w;
        }
    }
}
// rows 128 r .. of A, its scales and D in block r of the pair (or the one block), rows 128 r .. of B there too, B's scales in every block
inline void mma_fp4_pair(Block *leader, bool nv, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    const uint32_t N = ((idesc >> 17) & 0x3Fu) << 3, M = ((idesc >> 24) & 0x1Fu) << 4, sa = (idesc >> 29) & 3u, sb = (idesc >> 4) & 3u;
    EMU_CHECK(leader->rank == 0 && M == 256 && N % 32 == 0 && N <= 256 && ((idesc >> 7) & 7u) == 1 && ((idesc >> 10) & 7u) == 1, "E2M1 operands, 256 rows, issued by the leader");
    EMU_CHECK(((idesc >> 23) & 1u) == (nv ? 0u : 1u) && (nv ? sa == 0 && sb == 0 : (sa & 1) == 0 && (sb & 1) == 0), "scale type and ids");
    const uint32_t dcol = d_tmem & 0xFFFF, ca = sfa & 0xFFFF, cb = sfb & 0xFFFF, per = nv ? 16 : 32;
    if (dcol + N > 512 || ca + 4 > 512 || cb + 8 > 512) { fail("block-scaled MMA outside tensor memory"); return; }
    for (uint32_t r = 0; r < 2; ++r) {
        Block *blk = leader->cluster[r];
        auto scale = [&](uint32_t col, uint32_t row, uint32_t group, uint32_t id) {
            return scale_value(nv, (blk->tmem[(row & 31) * 512 + col + (row >> 5)] >> (8 * (id + group))) & 0xFF);
        };
        std::vector<float> a(128 * 64), b(N * 64);
        for (uint32_t i = 0; i < 128; ++i)
            for (uint32_t k = 0; k < 64; ++k) a[i * 64 + k] = fp4_operand(blk, a_desc, i, k) * scale(ca, i, k / per, sa);
        for (uint32_t i = 0; i < N; ++i)
            for (uint32_t k = 0; k < 64; ++k) b[i * 64 + k] = fp4_operand(leader->cluster[i / (N / 2)], b_desc, i % (N / 2), k) * scale(cb, i, k / per, sb);
        for (uint32_t m = 0; m < 128; ++m)
            for (uint32_t n = 0; n < N; ++n) {
                double acc = accumulate ? (double)__uint_as_float(blk->tmem[m * 512 + dcol + n]) : 0.0;
                for (uint32_t k = 0; k < 64; ++k) acc += (double)a[m * 64 + k] * b[n * 64 + k];
                blk->tmem[m * 512 + dcol + n] = __float_as_uint((float)acc);
            }
    }
}
inline void mma_fp4(Block *blk, bool nv, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    const uint32_t N = ((idesc >> 17) & 0x3Fu) << 3, M = ((idesc >> 24) & 0x1Fu) << 4, sa = (idesc >> 29) & 3u, sb = (idesc >> 4) & 3u;
    EMU_CHECK(M == 128 && ((idesc >> 7) & 7u) == 1 && ((idesc >> 10) & 7u) == 1, "E2M1 operands, 128 rows");
    EMU_CHECK(((idesc >> 23) & 1u) == (nv ? 0u : 1u), "scale type");
    EMU_CHECK(nv ? sa == 0 && sb == 0 : (sa & 1) == 0 && (sb & 1) == 0, "scale ids");
    EMU_CHECK(((a_desc >> 61) & 7u) == 2 && ((b_desc >> 61) & 7u) == 2, "128-byte swizzle");
    const uint32_t dcol = d_tmem & 0xFFFF, ca = sfa & 0xFFFF, cb = sfb & 0xFFFF;
    if (dcol + N > 512 || ca + 4 > 512 || cb + (N + 31) / 32 > 512) { fail("block-scaled MMA outside tensor memory"); return; }
    const uint32_t per = nv ? 16 : 32;
    auto scale = [&](uint32_t col, uint32_t row, uint32_t group, uint32_t id) {
        return scale_value(nv, (blk->tmem[(row & 31) * 512 + col + (row >> 5)] >> (8 * (id + group))) & 0xFF);
    };
    std::vector<float> a(128 * 64), b(N * 64);
    for (uint32_t r = 0; r < 128; ++r)
        for (uint32_t k = 0; k < 64; ++k) a[r * 64 + k] = fp4_operand(blk, a_desc, r, k) * scale(ca, r, k / per, sa);
    for (uint32_t r = 0; r < N; ++r)
        for (uint32_t k = 0; k < 64; ++k) b[r * 64 + k] = fp4_operand(blk, b_desc, r, k) * scale(cb, r, k / per, sb);
    for (uint32_t m = 0; m < 128; ++m)
        for (uint32_t n = 0; n < N; ++n) {
            double acc = accumulate ? (double)__uint_as_float(blk->tmem[m * 512 + dcol + n]) : 0.0;
            for (uint32_t k = 0; k < 64; ++k) acc += (double)a[m * 64 + k] * b[n * 64 + k];
            blk->tmem[m * 512 + dcol + n] = __float_as_uint((float)acc);
        }
}
}  // namespace emu

// Threads of the warps from this one on come so many milliseconds late to their first look at a barrier (-1 = none)
namespace emu {
inline std::atomic<int> g_late_warp{-1}, g_late_ms{0};
inline void come_late() {
    static thread_local bool been = false;
    if (been || g_late_warp.load() < 0 || (int)(threadIdx.x >> 5) < g_late_warp.load()) return;
    been = true;
    std::this_thread::sleep_for(std::chrono::milliseconds(g_late_ms.load()));
}
}  // namespace emu
extern "C" inline __attribute__((used, visibility("default"))) void emu_late_warps(int first, int ms) { emu::g_late_warp = first, emu::g_late_ms = ms; }
static inline bool mbar_test(uint32_t bar, uint32_t parity) {
    emu::come_late();
    return mbar_try(bar, parity);
}
static inline bool mbar_test_acquire_cluster(uint32_t bar, uint32_t parity) { return mbar_test(bar, parity); }
static inline void mbar_arrive_release_cluster(uint32_t cluster_addr) { mbar_arrive(cluster_addr); }
static inline void tc_cp_scales(uint32_t taddr, uint64_t desc) {
    if (emu::tc_deferred()) emu::tc_push([=] { emu::cp_scales(emu::g_block, taddr, desc); });
    else emu::cp_scales(emu::g_block, taddr, desc);
}
template <bool NV>
static inline void tc_mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (emu::tc_deferred()) emu::tc_push([=] { emu::mma_fp4(emu::g_block, NV, d, a, b, idesc, sfa, sfb, accumulate); });
    else emu::mma_fp4(emu::g_block, NV, d, a, b, idesc, sfa, sfb, accumulate);
}

static inline void tc_cp_scales_pair(uint32_t taddr, uint64_t desc) {
    auto both = [=] { for (int r = 0; r < 2; ++r) emu::cp_scales(emu::g_block->cluster[r], taddr, desc); };
    if (emu::tc_deferred()) emu::tc_push(both);
    else both();
}
template <bool NV>
static inline void tc_mma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (emu::tc_deferred()) emu::tc_push([=] { emu::mma_fp4_pair(emu::g_block, NV, d, a, b, idesc, sfa, sfb, accumulate); });
    else emu::mma_fp4_pair(emu::g_block, NV, d, a, b, idesc, sfa, sfb, accumulate);
}

// tcgen05.mma kind::f16 with f16 operands: A from tensor memory, B K-major in shared memory with the 128-byte swizzle
namespace emu {
inline void mma_ts_f16(Block *blk, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    const uint32_t N = ((idesc >> 17) & 0x3Fu) << 3, M = ((idesc >> 24) & 0x1Fu) << 4, dcol = d_tmem & 0xFFFF, acol = a_tmem & 0xFFFF;
    EMU_CHECK(M == 128 && N % 16 == 0 && N >= 16 && N <= 256 && ((idesc >> 4) & 3u) == 1 && ((idesc >> 7) & 7u) == 0 && ((idesc >> 10) & 7u) == 0, "D f32, A and B f16");
    EMU_CHECK(((b_desc >> 61) & 7u) == 2 && ((b_desc >> 46) & 1u) == 1, "128-byte swizzle, descriptor version 1");
    if (dcol + N > 512 || acol + 8 > 512) { fail("tcgen05.mma operands outside tensor memory"); return; }
    std::vector<float> b((size_t)N * 16);
    for (uint32_t n = 0; n < N; ++n)
        for (uint32_t k = 0; k < 16; ++k) {
            uint16_t h;
            memcpy(&h, smem_ptr(swizzle((smem_u32(blk->dyn) | desc_start(b_desc)) + (n >> 3) * desc_stride(b_desc) + (n & 7) * 128 + k * 2, 128)), 2);
            b[n * 16 + k] = (float)emu_f16_of(h);
        }
    for (uint32_t m = 0; m < 128; ++m)
        for (uint32_t n = 0; n < N; ++n) {
            double acc = accumulate ? (double)__uint_as_float(blk->tmem[m * 512 + dcol + n]) : 0.0;
            for (uint32_t k = 0; k < 16; ++k) {
                const uint32_t w = blk->tmem[m * 512 + acol + (k >> 1)];
                acc += (double)emu_f16_of(k & 1 ? w >> 16 : w & 0xFFFF) * (double)b[n * 16 + k];
            }
            blk->tmem[m * 512 + dcol + n] = __float_as_uint((float)acc);
        }
}
}  // namespace emu
static inline void tc_mma_ts_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (emu::tc_deferred()) emu::tc_push([=] { emu::mma_ts_f16(emu::g_block, d, a, b, idesc, accumulate); });
    else emu::mma_ts_f16(emu::g_block, d, a, b, idesc, accumulate);
}

// half of tensor memory: the model's allocation is the whole of it
static inline void tc_alloc_256(uint32_t result_smem) { tc_alloc_512(result_smem); }
static inline void tc_dealloc_256(uint32_t) {}
static inline void tc_st16(uint32_t taddr, const uint32_t *r) {
    const uint32_t lane = (taddr >> 16) + (threadIdx.x & 31), col = taddr & 0xFFFF;
    if (!(lane < 128 && col + 16 <= 512)) { emu::fail("tcgen05.st outside tensor memory"); return; }
    EMU_CHECK((taddr >> 16) == 32 * ((threadIdx.x >> 5) & 3), "a warp may only touch the lane quadrant warp % 4");
    for (int i = 0; i < 16; ++i) emu::g_block->tmem[lane * 512 + col + i] = r[i];
}
