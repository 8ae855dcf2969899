// The last of several workgroups to have stored its part adds them up, in the same launch.
//
// Parts are stored and read by relaxed atomics of agent scope, which go past the caches that one XCD does not share with
// the others.  last_to_arrive waits until a wave's stores have been acknowledged, a barrier makes that the whole
// workgroup's, and only then counts the workgroup: whoever counts last finds every part in memory.  The count goes back to 0,
// so that tickets are 0 between launches.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace prom {

#ifdef __HIPCC__
// Called by whole workgroups behind their stores; `shared` is a word of LDS.
__device__ __forceinline__ bool last_to_arrive(uint32_t* ticket, uint32_t of, uint32_t* shared) {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == of - 1) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = before;
  }
  __syncthreads();
  const bool last = *shared == of - 1;
  asm volatile("" ::: "memory");
  return last;
}
#endif

}  // namespace prom
