// Loads from device memory that go to LDS past the registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rtg {

// Lane i's 16 bytes at base + voff go to LDS lds + 16 i (the kernel waits itself).
// A load to LDS needs a wait state behind the write of M0; nobody adds it within
// an asm block.
__device__ __forceinline__ void load_lds16(unsigned voff, const void* base, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory", "m0");
}
// This wave's loads have landed, then the barrier.
__device__ __forceinline__ void wait_and_sync() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

}  // namespace rtg
