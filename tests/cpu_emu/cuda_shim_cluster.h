// Stand-ins for shrew_b200/csrc/ptx_cluster.cuh, beside cuda_shim_tcgen05_pair.h.  TEST INFRASTRUCTURE ONLY.
#pragma once

static inline void st_cluster_u32(uint32_t addr, uint32_t v) { memcpy(emu::smem_ptr(addr), &v, 4); }
