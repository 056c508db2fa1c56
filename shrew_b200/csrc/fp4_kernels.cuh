// Quantization to 4-bit microscaled floating point and back, sm_100a.
//
// A row of K values is cut into blocks, each with one scale; the codes are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//   MX: blocks of 32, scale 2^e as an E8M0 byte (e + 127, 255 = NaN):    e = max(floor(log2 amax) - 2, -127)
//   NV: blocks of 16, scale as an E4M3 byte, one f32 scale g a tensor:   s = e4m3(min(max(amax / (6 g), 2^-9), 448))
// where amax is the block's largest magnitude; a block of zeros gets the scale 1, a block with an infinity or a NaN the scale NaN
// (and codes 0), so that it comes back as NaN.  code = e2m1(x / scale), to nearest, ties to even, saturating; value = code * scale.
// Unless it is given, g is the smallest power of two with amax of the tensor (finite values) <= 448 * 6 * g: a power of two costs
// nothing of the scales' precision (they are floating point) and makes x / g exact.
//
// Every decision is the one exact arithmetic would take.  MX: x * 2^-e is exact.  NV: amax / 6 rounded to f32 never lands on a
// border of E4M3 that amax / 6 itself is not on (an f32 next to 6 times the border is more than half an ulp of the quotient away),
// and x / s is rounded once: q = x r with r = 1 / s rounded, corrected by the exact remainder, q + (x - q s) r (Markstein 1990), which by
// the same argument lands on a tie between codes only when x / s does.  tests/ compares with exact arithmetic, ties among the inputs.
//
// Layout: rows padded to whole 32s: codes [rows][Kp / 2] bytes, the even column in the low nibble; scales [rows][Kp / 32] (MX) or
// [rows][Kp / 16] (NV) bytes.  Padding has code 0 and, where a block is all padding, scale 1.
//
// Memory-bound: 2 or 4 bytes a value in and 0.53 or 0.56 out (the reverse in dequantization).  A thread takes 8 consecutive values
// (one or two 16-byte loads: four lanes are an MX block, two an NV block, so a block's maximum is two shuffles or one) and writes one
// word of codes.
//
// Device code only (no launch syntax; PTX behind ptx_fp4.cuh and ptx_small.cuh): also compiles for the CPU tests (tests/cpu_emu/).
#pragma once

#include "ptx_fp4.cuh"
#include "ptx_small.cuh"

namespace shrewq {
namespace {

constexpr int kFp4Threads = 256;
constexpr uint32_t kE4m3One = 0x38, kE4m3Nan = 0x7F, kE8m0One = 127, kE8m0Nan = 255;

// Eight values of a thread.  load_vec8: 16-byte aligned (32 for f32); load_guarded8: element by element, zero beyond `left`.
template <typename T>
__device__ __forceinline__ void load_vec8(const T *p, float *v);
template <>
__device__ __forceinline__ void load_vec8<float>(const float *p, float *v) {
    uint32_t r[8];
    ld_stream_32(p, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void load_vec8<__nv_bfloat16>(const __nv_bfloat16 *p, float *v) {
    const uint4 w = ld_once_16(p);
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
}
template <>
__device__ __forceinline__ void load_vec8<__half>(const __half *p, float *v) {
    const uint4 w = ld_once_16(p);
    f32x2_of_f16x2(w.x, v[0], v[1]);
    f32x2_of_f16x2(w.y, v[2], v[3]);
    f32x2_of_f16x2(w.z, v[4], v[5]);
    f32x2_of_f16x2(w.w, v[6], v[7]);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ void load_guarded8(const T *p, size_t left, float *v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (size_t)i < left ? to_f32(p[i]) : 0.0f;
}

// The tensor scale that an amax asks for: the smallest power of two g with 2688 g >= amax (2688 = 448 * 6)
__device__ __forceinline__ float fp4_tensor_scale(float amax) {
    if (!(amax > 0.0f)) return 1.0f;
    const uint32_t b = __float_as_uint(__fdiv_rn(amax, 2688.0f));
    uint32_t e = (b >> 23) + ((b & 0x7FFFFFu) ? 1u : 0u);
    e = e < 1u ? 1u : e;
    return __uint_as_float(e << 23);
}

// a / 6 and 1 / s, rounded to nearest: an approximation and one step with its exact remainder (Markstein 1990: right for every a whose quotient is a
// normal number, and smaller ones end at the least scale; s runs through the 126 values that a scale can have, and tests/test_gpu_fp4_exact.py
// through all of them, with every border of their codes).  3 instructions each.
__device__ __forceinline__ float div6_rn(float a) {
    const float r = 0.166666672f, q = a * r;  // r = 1/6 rounded to nearest
    return __fmaf_rn(__fmaf_rn(-6.0f, q, a), r, q);
}
__device__ __forceinline__ float recip_e4m3_rn(float s) {
    const float r = recip_approx(s);
    return __fmaf_rn(__fmaf_rn(-s, r, 1.0f), r, r);
}

// One thread's part of a block: v[8] -> a word of codes and the block's scale byte (the same in all lanes of the block).  Every lane of
// the warp takes part in the shuffles.  GIVEN (NV): a tensor scale that was not found from the tensor may take finite values beyond f32; they
// saturate.  (A scale that was found does not, and the test for it costs 2 of 62 us in the round trip of 11008 x 4096.)
template <bool NV, bool GIVEN>
__device__ __forceinline__ uint32_t fp4_encode(float *v, float inv_g, uint32_t &byte) {
    auto scale_values = [&] {
#pragma unroll
        for (int i = 0; i < 8; i += 2) mul_f32x2(v[i], v[i + 1], inv_g, v[i], v[i + 1]);
    };
    if constexpr (NV && !GIVEN) scale_values();
    float amax = max_abs_nan(v[0], v[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) amax = max_abs_nan(amax, max_abs_nan(v[i], v[i + 1]));
    amax = max_abs_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    if constexpr (!NV) amax = max_abs_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    const float inf = __uint_as_float(0x7F800000u);
    const bool bad = !(amax < inf);
    if constexpr (NV) {
        if constexpr (GIVEN) {
            amax *= inv_g;  // (what the largest of the products below is: rounding keeps their order)
            scale_values();
            if (amax == inf && !bad) {
                const float most = __uint_as_float(0x7F7FFFFFu);
                amax = most;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -most), most);
            }
        }
        byte = amax == 0.0f ? kE4m3One : cvt_e4m3(fminf(fmaxf(div6_rn(amax), 0.001953125f), 448.0f));
        float s, unused;
        f32x2_of_f16x2(cvt_f16x2_e4m3(byte), s, unused);
        const float r = recip_e4m3_rn(s);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float q0, q1, e0, e1;
            mul_f32x2(v[i], v[i + 1], r, q0, q1);
            fma_f32x2(q0, q1, -s, v[i], v[i + 1], e0, e1);
            fma_f32x2(e0, e1, r, q0, q1, v[i], v[i + 1]);
        }
        if (bad) byte = kE4m3Nan;
    } else {
        const int e = (int)(__float_as_uint(amax) >> 23) - 2;
        byte = amax == 0.0f ? kE8m0One : (uint32_t)(e > 0 ? e : 0);
        const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
        for (int i = 0; i < 8; i += 2) mul_f32x2(v[i], v[i + 1], inv, v[i], v[i + 1]);
        if (bad) byte = kE8m0Nan;
    }
    return bad ? 0u : cvt_e2m1x8(v);
}

__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
    return __uint_as_float(b == 0 ? 0x00400000u : b == 255u ? 0x7FFFFFFFu : b << 23);
}

// ---- the tensor's scale (NV where it is not given) ------------------------------------------------------------------------------
// The scale that the largest finite magnitude asks for is the largest of the scales that the magnitudes of parts ask for, since it grows with the
// magnitude; 0 stands for a part of zeros.  The memory is the call's own, so that calls on other streams and replays of captured ones cannot meet:
// either a word behind g for every block, of which each block of the quantizing kernel takes the maximum, or g alone, which is 0 before and
// which the blocks raise (positive floats are ordered as their words are): a launch more, for the zero.  One block writes g as it is.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kFp4Threads)
fp4_tensor_scale_kernel(const T *x, size_t rows, size_t cols, size_t ld, float *g, int parts) {
    pdl_launch_dependents();
    pdl_wait();
    float amax = 0.0f;
    const float inf = __uint_as_float(0x7F800000u);
    auto take = [&](const float *v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = fabsf(v[i]);
            amax = fmaxf(amax, a < inf ? a : 0.0f);
        }
    };
    const size_t per_row = (cols + 7) / 8, total = FLAT ? rows * cols / 8 : rows * per_row;
    const size_t step = (size_t)gridDim.x * kFp4Threads;
    size_t i = (size_t)blockIdx.x * kFp4Threads + threadIdx.x;
    if constexpr (FLAT) {
        constexpr int U = sizeof(T) == 2 ? 8 : 4;  // 128 bytes a thread under way, the end of the tensor included
        for (; i < total; i += U * step) {
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u * step < total) load_vec8<T>(x + (i + u * step) * 8, v[u]);
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) take(v[u]);
        }
    }
    for (; !FLAT && i < total; i += step) {
        float v[8];
        const size_t row = i / per_row, c = (i % per_row) * 8;
        load_guarded8<T>(x + row * ld + c, cols - c, v);
        take(v);
    }
    __shared__ float s_max[kFp4Threads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kFp4Threads / 32; ++w) amax = fmaxf(amax, s_max[w]);
        const float mine = amax > 0.0f ? fp4_tensor_scale(amax) : 0.0f;
        if (parts) g[1 + blockIdx.x] = mine;
        else if (gridDim.x == 1) *g = mine;
        else if (mine > 0.0f) atomicMax(reinterpret_cast<unsigned int *>(g), __float_as_uint(mine));
    }
}

// The tensor scale for every thread of a block.  source: kScaleGiven, read; else found by the kernel before, and 1 where that found nothing but
// zeros: kScaleFound in g itself (block 0 then writes the 1; who reads the word before and who reads it after takes it for 1 alike), else in as
// many words behind g (block 0 writes g).
constexpr int kScaleGiven = 0, kScaleFound = -1;
__device__ __forceinline__ float fp4_read_tensor_scale(float *g, int source, int threads) {
    if (source <= 0) {
        const float v = __uint_as_float((uint32_t)ld_written_s32(reinterpret_cast<const int *>(g)));
        if (source == kScaleGiven || v != 0.0f) return v;
        if (blockIdx.x == 0 && threadIdx.x == 0) *g = 1.0f;
        return 1.0f;
    }
    __shared__ float s_part[32];
    float m = 0.0f;
    for (int i = threadIdx.x; i < source; i += threads) m = fmaxf(m, g[1 + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = s_part[0];
    for (int w = 1; w < threads / 32; ++w) m = fmaxf(m, s_part[w]);
    m = m == 0.0f ? 1.0f : m;
    if (blockIdx.x == 0 && threadIdx.x == 0) *g = m;
    return m;
}

// ---- quantize: rows that are whole aligned 32s, one after the other: a flat stream of groups of 8 ------------------------------
// U groups a thread, requested before the first is used (and before the tensor's scale is put together, which costs a block some 2000 cycles where
// it is in parts, so that the grid is no more than what is resident then).  Where a pass before this one has found the scale, reading the tensor
// from the front (not GIVEN), the chunks go through it from its end: what that pass left in L2 is read first.
template <typename T, bool NV, bool GIVEN, int U>
__global__ void __launch_bounds__(kFp4Threads)
fp4_quantize_flat_kernel(const T *x, size_t groups, float *g, int source, uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t chunks = (groups + kFp4Threads * U - 1) / (kFp4Threads * U);
    float v[U][8];
    auto load = [&](size_t base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t i = base + (size_t)u * kFp4Threads;
            if (i < groups) load_vec8<T>(x + i * 8, v[u]);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
            }
        }
    };
    auto base_of = [&](size_t chunk) { return (GIVEN ? chunk : chunks - 1 - chunk) * (size_t)(kFp4Threads * U) + threadIdx.x; };
    load(base_of(blockIdx.x));
    float inv_g = 1.0f;
    if constexpr (NV) inv_g = __fdiv_rn(1.0f, fp4_read_tensor_scale(g, source, kFp4Threads));
    for (size_t chunk = blockIdx.x;;) {
        const size_t base = base_of(chunk);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t i = base + (size_t)u * kFp4Threads;
            uint32_t byte;
            const uint32_t word = fp4_encode<NV, GIVEN>(v[u], inv_g, byte);
            if (i < groups) {
                codes[i] = word;
                if constexpr (NV) {
                    if ((i & 1) == 0) scales[i >> 1] = (uint8_t)byte;
                } else {
                    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
                }
            }
        }
        chunk += gridDim.x;
        if (chunk >= chunks) break;
        load(base_of(chunk));
    }
}

// Byte offset of the scale of (row, block) in the order that the block-scaled matrix instructions read: pieces of 128 rows by 4
// blocks, 512 bytes each, k fastest; inside a piece row r sits at (r % 32) * 16 + (r / 32) * 4.  `pieces`: pieces along a row.
__device__ __forceinline__ size_t scale_piece_offset(size_t row, size_t block, size_t pieces) {
    return ((row >> 7) * pieces + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// ---- quantize: any rows (strides, widths, alignments) ---------------------------------------------------------------------------
// A CTA a row at a time.  vec_ok: rows start on 16-byte (f32: 32-byte) boundaries.
template <typename T, bool NV>
__global__ void __launch_bounds__(kFp4Threads)
fp4_quantize_rows_kernel(const T *x, size_t rows, size_t cols, size_t ld, int vec_ok, float *g, int source, size_t blocks_out,
                         uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    pdl_launch_dependents();
    pdl_wait();
    float inv_g = 1.0f;
    if constexpr (NV) inv_g = __fdiv_rn(1.0f, fp4_read_tensor_scale(g, source, (int)blockDim.x));
    constexpr int kShift = NV ? 1 : 2;                  // groups of 8 in a block, as a power of two
    const size_t words = (cols + 31) / 32 * 4;          // words of codes in a row
    const size_t groups = blocks_out << kShift;         // >= words
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *src = x + row * ld;
        for (size_t i0 = 0; i0 < groups; i0 += blockDim.x) {  // (uniform: the shuffles need whole warps)
            const size_t i = i0 + threadIdx.x;
            float v[8];
            if (vec_ok && i * 8 + 8 <= cols) load_vec8<T>(src + i * 8, v);
            else load_guarded8<T>(src + i * 8, i * 8 < cols ? cols - i * 8 : 0, v);
            uint32_t byte;
            const uint32_t word = fp4_encode<NV, true>(v, inv_g, byte);
            if (i < words) codes[row * words + i] = word;
            if (i < groups && (i & ((1 << kShift) - 1)) == 0) scales[row * blocks_out + (i >> kShift)] = (uint8_t)byte;
        }
    }
}

// ---- quantize: the activations of a 4-bit product --------------------------------------------------------------------------------
// As above, but the scales go to the order of scale_piece_offset, out to whole pieces (scale 1 beyond the row's end): `units` runs of 256
// values a row, a warp a run, two of them requested together.  Four blocks of a row are one word of a piece.  Indices within a row are 32-bit and
// whole runs take no guards: with the indexing of the kernel above 4096 x 11008 bf16 took 130 instructions for 8 values a lane and 37 us.
template <typename T, bool NV>
__global__ void __launch_bounds__(kFp4Threads)
fp4_quantize_acts_kernel(const T *x, size_t rows, uint32_t cols, int vec_ok, const float *g_in, uint32_t units, uint32_t *__restrict__ codes,
                         uint8_t *__restrict__ scales) {
    pdl_launch_dependents();
    pdl_wait();
    float inv_g = 1.0f;
    if constexpr (NV) inv_g = __fdiv_rn(1.0f, *g_in);
    constexpr int kShift = NV ? 1 : 2, kPieces = NV ? 4 : 2;  // groups of 8 in a block, as a power of two; pieces that a run fills
    const uint32_t words = (cols + 31) / 32 * 4, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const size_t pieces = (size_t)units * kPieces;
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *src = x + row * cols;
        uint32_t *code_row = codes + row * words;
        uint8_t *scale_row = scales + scale_piece_offset(row, 0, pieces) + (lane >> (kShift + 2)) * 512;
        for (uint32_t u = threadIdx.x >> 5; u < units; u += 2 * warps) {
            float v[2][8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t i = (u + k * warps) * 32 + lane;
                if (k == 1 && u + warps >= units) break;
                if (vec_ok && (u + k * warps + 1) * 256 <= cols) load_vec8<T>(src + (size_t)i * 8, v[k]);
                else load_guarded8<T>(src + (size_t)i * 8, i * 8 < cols ? cols - i * 8 : 0, v[k]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t run = u + k * warps, i = run * 32 + lane;
                if (k == 1 && run >= units) break;
                uint32_t byte;
                const uint32_t word = fp4_encode<NV, true>(v[k], inv_g, byte);
                if (i < words) code_row[i] = word;
                uint32_t four = byte | __shfl_xor_sync(0xFFFFFFFFu, byte, 1 << kShift) << 8;
                four |= __shfl_xor_sync(0xFFFFFFFFu, four, 2 << kShift) << 16;
                if ((lane & ((4 << kShift) - 1)) == 0) *reinterpret_cast<uint32_t *>(scale_row + (size_t)run * (kPieces * 512)) = four;
            }
        }
    }
}

// ---- dequantize ----------------------------------------------------------------------------------------------------------------
// eight codes and their scale -> eight f32: code * s exactly (three bits by one or four), then * g, rounded once
template <bool NV>
__device__ __forceinline__ void fp4_decode(uint32_t word, uint32_t byte, float g, float *v) {
    uint32_t h[4];
    cvt_f16x8_e2m1(word, h);
    float s, unused;
    if constexpr (NV) f32x2_of_f16x2(cvt_f16x2_e4m3(byte), s, unused);
    else s = e8m0_to_f32(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f32x2_of_f16x2(h[i], v[2 * i], v[2 * i + 1]);
        v[2 * i] *= s;
        v[2 * i + 1] *= s;
        if constexpr (NV) {
            v[2 * i] *= g;
            v[2 * i + 1] *= g;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store_vec8(T *p, const float *v);
template <>
__device__ __forceinline__ void store_vec8<float>(float *p, const float *v) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[i]);
    st_32(p, r);
}
template <>
__device__ __forceinline__ void store_vec8<__nv_bfloat16>(__nv_bfloat16 *p, const float *v) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2_rn(v[1], v[0]), pack_bf16x2_rn(v[3], v[2]), pack_bf16x2_rn(v[5], v[4]),
                                               pack_bf16x2_rn(v[7], v[6]));
}
template <>
__device__ __forceinline__ void store_vec8<__half>(__half *p, const float *v) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_f16x2_rn(v[1], v[0]), pack_f16x2_rn(v[3], v[2]), pack_f16x2_rn(v[5], v[4]),
                                               pack_f16x2_rn(v[7], v[6]));
}
__device__ __forceinline__ void from_f32(float v, float *p) { *p = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half *p) { *p = __float2half_rn(v); }

// flat: rows that are whole 32s and an aligned output; U groups of 8 a thread
template <typename T, bool NV, int U>
__global__ void __launch_bounds__(kFp4Threads)
fp4_dequantize_flat_kernel(const uint32_t *codes, const uint8_t *scales, const float *g_in, size_t groups, T *__restrict__ out) {
    pdl_launch_dependents();
    pdl_wait();
    const float g = NV ? *g_in : 1.0f;
    const size_t base = (size_t)blockIdx.x * (kFp4Threads * U) + threadIdx.x;
    uint32_t word[U], byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const size_t i = base + (size_t)u * kFp4Threads;
        word[u] = i < groups ? __ldcs(codes + i) : 0u;
        byte[u] = i < groups ? scales[i >> (NV ? 1 : 2)] : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const size_t i = base + (size_t)u * kFp4Threads;
        if (i >= groups) break;
        float v[8];
        fp4_decode<NV>(word[u], byte[u], g, v);
        store_vec8<T>(out + i * 8, v);
    }
}

template <typename T, bool NV>
__global__ void __launch_bounds__(kFp4Threads)
fp4_dequantize_rows_kernel(const uint32_t *codes, const uint8_t *scales, const float *g_in, size_t rows, size_t cols,
                           int vec_ok, T *__restrict__ out) {
    pdl_launch_dependents();
    pdl_wait();
    const float g = NV ? *g_in : 1.0f;
    const size_t per_row = (cols + 7) / 8, words = (cols + 31) / 32 * 4;
    const size_t total = rows * per_row;
    for (size_t i = (size_t)blockIdx.x * kFp4Threads + threadIdx.x; i < total; i += (size_t)gridDim.x * kFp4Threads) {
        const size_t row = i / per_row, c = i % per_row;
        float v[8];
        fp4_decode<NV>(codes[row * words + c], scales[(row * words + c) >> (NV ? 1 : 2)], g, v);
        T *dst = out + row * cols + c * 8;
        if (vec_ok && c * 8 + 8 <= cols) store_vec8<T>(dst, v);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c * 8 + j < cols) from_f32(v[j], dst + j);
    }
}

}  // namespace
}  // namespace shrewq
