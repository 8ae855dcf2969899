// Transfers from memory to LDS that pass no registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace prom {

#ifdef __HIPCC__
typedef int BufferWords __attribute__((ext_vector_type(4)));

// 16 bytes a lane from `off` (and `base`, the same for all lanes) within the buffer to LDS at `to` + 16 * lane; `to` is
// uniform.  A transfer may read m0 one wait state after it is written and no sooner, and the compiler does not look into
// a block of assembly for that: s_nop.
__device__ __forceinline__ void lds_from_buffer(uint32_t to, uint32_t off, BufferWords buffer) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(buffer)
               : "memory", "m0");
}
__device__ __forceinline__ void lds_from_buffer(uint32_t to, uint32_t off, BufferWords buffer, int base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(buffer),
               "s"(base)
               : "memory", "m0");
}
#endif

}  // namespace prom
