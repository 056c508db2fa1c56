// Cluster instructions for kernels whose cluster size is chosen at launch (the cluster's barrier and address mapping come from
// ptx_tcgen05_pair.cuh).  The CPU tests (tests/cpu_emu/) provide stand-ins.
#pragma once

#include "ptx_tcgen05_pair.cuh"

#ifndef SHREWQ_CPU_EMU
namespace shrewq {
namespace {

// store into the shared memory of a CTA of the cluster (address from map_to_cta)
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

}  // namespace
}  // namespace shrewq
#endif  // SHREWQ_CPU_EMU
