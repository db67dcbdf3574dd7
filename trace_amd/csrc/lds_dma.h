// LDS-DMA helpers shared by the kernels that stage tiles through an LDS ring (gfx950).
#pragma once
#include "common.h"

namespace trace {

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

__device__ __forceinline__ void glds16(const void* g, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((gptr_t)g, (lptr_t)lds_wave_base, 16, 0, 0);
}
// The same with the NON-TEMPORAL cache policy (aux bit 1 = nt on gfx940+): for operands streamed from HBM exactly once -
// the weights of the 100352-wide FCs.  A plain load allocates in the memory-side cache and, behind kernels that
// wrote, pays for the write-back of the dirty lines it evicts: tools/stream_probe.hip reads fc1's 616 MB at 3.4 TB/s
// with plain loads behind a writer (6.1 TB/s on clean caches) and at 6.8 TB/s with nt loads in either state.
__device__ __forceinline__ void glds16_nt(const void* g, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((gptr_t)g, (lptr_t)lds_wave_base, 16, 0, 2);
}

template <int N> __device__ __forceinline__ void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// The barrier of the LDS rings.  A wave must not ARRIVE with LDS reads still in flight: behind the barrier the other
// waves refill - by LDS-DMA - the very stage those reads came from (write-after-read).  `__builtin_amdgcn_s_barrier()`
// alone does not order them: hipcc keeps a stage's last fragment reads in flight across it and waits for them
// (`s_waitcnt lgkmcnt`) only in front of the MFMAs that it sank below the barrier.  Alone on a CU the reads always win the
// race against a refill that still has an L2 round trip ahead of it; beside another kernel's workgroups that keep the CU's
// LDS pipeline busy (a second stream or a forked graph branch) the refill can land first and the MFMA consumes bytes of
// the NEXT K-step: one wrong 32-position wave column per ~10^5 workgroups (tools/race_probe.py names the launch,
// tools/scan_barrier_hazard.py lists every kernel whose assembly had the pattern).
__device__ __forceinline__ void ring_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace trace
