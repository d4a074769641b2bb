// paged_dev.h -- device functions that the paged cache's kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// One 64-bit word of host-mapped memory: (code, argument), the first one kept.
__device__ __forceinline__ void paged_err(uint64_t* __restrict__ err, uint32_t code, uint32_t arg) {
  if (__hip_atomic_load(err, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == 0u)
    __hip_atomic_store(err, ((uint64_t)arg << 32) | code, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Every store of this wave is where the agent's other workgroups see it, before anything
// that follows: relaxed stores alone would leave the compiler free to move them behind the
// wait, and a release at agent scope writes back a whole L2.
__device__ __forceinline__ void stores_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
}

// sum over the lanes up to this one: within rows of 16, then across them
__device__ __forceinline__ uint32_t scan64_lanes(uint32_t v) {
#define SCAN_DPP(CTRL, ROWS) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false)
  SCAN_DPP(0x111, 0xF);  // row_shr 1, 2, 4, 8
  SCAN_DPP(0x112, 0xF);
  SCAN_DPP(0x114, 0xF);
  SCAN_DPP(0x118, 0xF);
  SCAN_DPP(0x142, 0xA);  // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
  SCAN_DPP(0x143, 0xC);
#undef SCAN_DPP
  return v;
}
