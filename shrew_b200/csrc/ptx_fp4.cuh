// The PTX instructions of the 4-bit floating point kernels (conversions, wide loads and stores), each behind a small function.
// The CPU tests (tests/cpu_emu/) provide stand-ins with the same names and semantics.
#pragma once

#ifndef SHREWQ_CPU_EMU
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace shrewq {
namespace {

// eight f32 -> eight E2M1 codes in a word, v[0] in the lowest nibble
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float *v) {
    uint32_t d;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(d)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}
// eight E2M1 codes (a word) -> four packed f16x2, exact; h[0] holds the two lowest codes
__device__ __forceinline__ void cvt_f16x8_e2m1(uint32_t w, uint32_t *h) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// one f32 -> E4M3 byte, round to nearest even, saturating at 448
__device__ __forceinline__ uint32_t cvt_e4m3(float v) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(0.0f), "f"(v));
    return d & 0xFFu;
}
// two E4M3 bytes (low half of a word) -> packed f16x2, exact
__device__ __forceinline__ uint32_t cvt_f16x2_e4m3(uint32_t two) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)two));
    return d;
}
__device__ __forceinline__ void f32x2_of_f16x2(uint32_t h, float &lo, float &hi) {
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}
// two f32 -> packed f16x2, round to nearest even
__device__ __forceinline__ uint32_t pack_f16x2_rn(float hi, float lo) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// max(|a|, |b|), NaN if either is
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
// max(v, 0), NaN for NaN
__device__ __forceinline__ float relu_nan(float v) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(v), "f"(0.0f));
    return d;
}
// 16 or 32 bytes, read once / written once.  Not through the read-only path: they may be what the kernel before in the stream writes, which may
// still run when this one is launched early.
__device__ __forceinline__ uint4 ld_once_16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void ld_stream_32(const void *p, uint32_t *r) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}
__device__ __forceinline__ void st_32(void *p, const uint32_t *r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// packed f16x2 product, round to nearest even, subnormals kept
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// packed bf16x2 product, round to nearest even
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t smem_offset(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// asynchronous copies global -> shared memory of this thread's own bytes (16, past L1; 4); `valid` false: zeros, nothing is read
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
// two f32 operations an instruction, rounded as the single ones: (a0, a1) * s, (a0, a1) * s + (c0, c1)
__device__ __forceinline__ void mul_f32x2(float a0, float a1, float s, float &d0, float &d1) {
    asm("{\n\t.reg .b64 a, s, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\t"
        "mul.rn.f32x2 d, a, s;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(s));
}
__device__ __forceinline__ void fma_f32x2(float a0, float a1, float s, float c0, float c1, float &d0, float &d1) {
    asm("{\n\t.reg .b64 a, s, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 c, {%5, %6};\n\t"
        "fma.rn.f32x2 d, a, s, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(s), "f"(c0), "f"(c1));
}
// 2^x and 1/x, good to a few ulp; results below 2^-126 are 0
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float recip_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// A word that the kernel before in the stream has written, read where it stands in the program, from L2.  (Through a const __restrict__ pointer
// it would be a load of data that never changes, which the compiler may move to before griddepcontrol.wait.)
__device__ __forceinline__ int ld_written_s32(const int *p) {
    int v;
    asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// this thread arrives on the barrier (of a count that includes it) when all of its copies so far have landed
__device__ __forceinline__ void copy_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest N groups of this thread have landed, visible to this thread
template <int N>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace shrewq
#endif  // SHREWQ_CPU_EMU
