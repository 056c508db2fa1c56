// Stand-ins for the PTX instructions of shrew_b200/csrc/ptx_fp4.cuh and the few intrinsics next to them, beside cuda_shim.h.
// TEST INFRASTRUCTURE ONLY.  The conversions are written from the formats' definitions: round to nearest, ties to even.
#pragma once
#include "cuda_shim.h"

namespace emu {
// address of a shared-memory offset that smem_u32 (cuda_shim_tcgen05.h, or below) made from a pointer into the block's dynamic memory
inline void *smem_ptr_of(uint32_t addr) {
    return reinterpret_cast<void *>((reinterpret_cast<uintptr_t>(g_block->dyn) & ~uintptr_t(0xFFFFFFFFu)) | addr);
}
}  // namespace emu
static inline uint32_t smem_offset(const void *p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }

static inline float __fdiv_rn(float a, float b) { return a / b; }
static inline float __frcp_rn(float a) { return 1.0f / a; }
static inline float rsqrtf(float a) { return (float)(1.0 / sqrt((double)a)); }

static inline uint32_t emu_e2m1(float v) {
    static const float grid[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    const uint32_t sign = (__float_as_uint(v) >> 31) << 3;
    const float a = fabsf(v);
    if (!(a < 6.0f)) return sign | 7u;
    uint32_t c = 0;
    while (grid[c + 1] <= a) ++c;
    const float lo = a - grid[c], hi = grid[c + 1] - a;
    return sign | (lo < hi || (lo == hi && (c & 1) == 0) ? c : c + 1);
}
static inline uint32_t cvt_e2m1x8(const float *v) {
    uint32_t d = 0;
    for (int i = 0; i < 8; ++i) d |= emu_e2m1(v[i]) << (4 * i);
    return d;
}
static inline uint32_t emu_f16_bits(float v) { _Float16 h = (_Float16)v; uint16_t u; memcpy(&u, &h, 2); return u; }
static inline float emu_f16_value(uint32_t bits) { uint16_t u = (uint16_t)bits; _Float16 h; memcpy(&h, &u, 2); return (float)h; }
static inline float emu_e2m1_value(uint32_t c) {
    static const float grid[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    return c & 8 ? -grid[c & 7] : grid[c & 7];
}
static inline void cvt_f16x8_e2m1(uint32_t w, uint32_t *h) {
    for (int i = 0; i < 4; ++i)
        h[i] = emu_f16_bits(emu_e2m1_value((w >> (8 * i)) & 15u)) | emu_f16_bits(emu_e2m1_value((w >> (8 * i + 4)) & 15u)) << 16;
}
static inline float emu_e4m3_value(uint32_t b) {
    const int e = (b >> 3) & 15, m = b & 7;
    const float v = (b & 0x7F) == 0x7F ? NAN : e ? ldexpf(1.0f + m / 8.0f, e - 7) : ldexpf(m / 8.0f, -6);
    return b & 0x80 ? -v : v;
}
static inline uint32_t cvt_e4m3(float v) {
    if (v != v) return 0x7F;
    const float a = fabsf(v);
    uint32_t c = 0;  // the nearest byte, ties to the even one, 448 at most
    while (c < 0x7E && emu_e4m3_value(c + 1) <= a) ++c;
    if (c < 0x7E) {
        const float lo = a - emu_e4m3_value(c), hi = emu_e4m3_value(c + 1) - a;
        if (lo > hi || (lo == hi && (c & 1))) ++c;
    }
    return c | (__float_as_uint(v) >> 31) << 7;
}
static inline uint32_t cvt_f16x2_e4m3(uint32_t two) { return emu_f16_bits(emu_e4m3_value(two & 0xFF)) | emu_f16_bits(emu_e4m3_value((two >> 8) & 0xFF)) << 16; }
static inline void f32x2_of_f16x2(uint32_t h, float &lo, float &hi) { lo = emu_f16_value(h & 0xFFFF); hi = emu_f16_value(h >> 16); }
static inline uint32_t pack_f16x2_rn(float hi, float lo) { return emu_f16_bits(hi) << 16 | emu_f16_bits(lo); }
static inline float max_abs_nan(float a, float b) { return a != a || b != b ? NAN : fmaxf(fabsf(a), fabsf(b)); }
static inline float relu_nan(float v) { return v != v ? NAN : fmaxf(v, 0.0f); }
static inline uint4 ld_once_16(const void *p) {
    EMU_CHECK((reinterpret_cast<uintptr_t>(p) & 15) == 0, "a 16-byte load off its boundary");
    uint4 v;
    memcpy(&v, p, 16);
    return v;
}
static inline void ld_stream_32(const void *p, uint32_t *r) {
    EMU_CHECK((reinterpret_cast<uintptr_t>(p) & 31) == 0, "a 32-byte load off its boundary");
    memcpy(r, p, 32);
}
static inline void st_32(void *p, const uint32_t *r) {
    EMU_CHECK((reinterpret_cast<uintptr_t>(p) & 31) == 0, "a 32-byte store off its boundary");
    memcpy(p, r, 32);
}
static inline uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    return pack_f16x2_rn(emu_f16_value(a >> 16) * emu_f16_value(b >> 16), emu_f16_value(a & 0xFFFF) * emu_f16_value(b & 0xFFFF));
}
static inline uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    return pack_bf16x2_rn(emu_f32_of_bf16(a >> 16) * emu_f32_of_bf16(b >> 16), emu_f32_of_bf16(a & 0xFFFF) * emu_f32_of_bf16(b & 0xFFFF));
}

// cp.async: performed when it is waited for, so that a read without a wait finds old bytes
namespace emu {
struct AsyncCopy { void *dst; uint8_t data[16]; int bytes; int group; };
inline thread_local std::vector<AsyncCopy> g_copies;
inline thread_local int g_copy_group = 0;
inline void copy_async(uint32_t dst, const void *src, int bytes, bool valid) {
    AsyncCopy c{smem_ptr_of(dst), {0}, bytes, g_copy_group};
    if (valid) memcpy(c.data, src, bytes);
    EMU_CHECK(!valid || (reinterpret_cast<uintptr_t>(src) % bytes) == 0, "cp.async off its boundary");
    g_copies.push_back(c);
}
}  // namespace emu
static inline void copy_async_16(uint32_t dst, const void *src, bool valid) { emu::copy_async(dst, src, 16, valid); }
static inline void copy_async_4(uint32_t dst, const void *src, bool valid) { emu::copy_async(dst, src, 4, valid); }
static inline void copy_async_commit() { ++emu::g_copy_group; }
template <int N>
static inline void copy_async_wait() {
    auto &v = emu::g_copies;
    size_t kept = 0;
    for (auto &c : v) {
        if (c.group < emu::g_copy_group - N) memcpy(c.dst, c.data, c.bytes);
        else v[kept++] = c;
    }
    v.resize(kept);
}
static inline void mul_f32x2(float a0, float a1, float s, float &d0, float &d1) { d0 = a0 * s, d1 = a1 * s; }
static inline void fma_f32x2(float a0, float a1, float s, float c0, float c1, float &d0, float &d1) {
    d0 = fmaf(a0, s, c0), d1 = fmaf(a1, s, c1);
}
static inline int ld_written_s32(const int *p) { return *p; }
static inline float exp2_approx(float x) { return exp2f(x); }
static inline float recip_approx(float x) { return 1.0f / x; }
static inline void mbar_arrive(uint32_t bar);
static inline void copy_async_arrive(uint32_t bar) {
    for (auto &c : emu::g_copies) memcpy(c.dst, c.data, c.bytes);
    emu::g_copies.clear();
    mbar_arrive(bar);
}
