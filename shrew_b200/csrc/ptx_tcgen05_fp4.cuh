// The PTX instructions of the block-scaled tensor-core kernels (tcgen05.mma kind::mxf4 / kind::mxf4nvf4, tcgen05.cp of their scales),
// each behind a small function; the rest comes from ptx_tcgen05.cuh.  The CPU tests (tests/cpu_emu/) provide stand-ins.
#pragma once

#include "ptx_tcgen05.cuh"

#ifndef SHREWQ_CPU_EMU
namespace shrewq {
namespace {

// 32 rows of 16 bytes in shared memory (rows 16 bytes apart) -> four columns of tensor memory, the same in all four lane quadrants
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[128 x N] (+)= (A[128 x 64] * scales a) * (B[N x 64] * scales b)^T, E2M1 operands from shared memory, scales from tensor memory.
// NV: E4M3 scales for blocks of 16 (four a row), else E8M0 for blocks of 32 (two a row)
template <bool NV>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (NV)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

}  // namespace
}  // namespace shrewq
#endif  // SHREWQ_CPU_EMU
