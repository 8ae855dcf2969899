// Joins over the 64 lanes of a wave, by DPP.
#pragma once

#include <hip/hip_runtime.h>

namespace prom {

#ifdef __HIPCC__
// v of another lane of the wave, 64 bits; 0 where there is none.
template <int kCtrl, int kRows>
__device__ __forceinline__ unsigned long long moved(unsigned long long v) {
  const int low = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRows, 0xF, false);
  const int high = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), kCtrl, kRows, 0xF, false);
  return (unsigned long long)(uint32_t)high << 32 | (uint32_t)low;
}
// The wave's v joined by `op`, whose neutral element is 0, in every lane: rows of sixteen by shifts of 1, 2, 4 and 8, then the
// rows by broadcasts of their last lanes.
template <typename F>
__device__ __forceinline__ unsigned long long wave_join(unsigned long long v, F&& op) {
  v = op(v, moved<0x111, 0xF>(v));
  v = op(v, moved<0x112, 0xF>(v));
  v = op(v, moved<0x114, 0xF>(v));
  v = op(v, moved<0x118, 0xF>(v));
  v = op(v, moved<0x142, 0xA>(v));
  v = op(v, moved<0x143, 0xC>(v));
  const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)v, 63);
  const uint32_t high = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63);
  return (unsigned long long)high << 32 | low;
}
__device__ __forceinline__ double wave_sum(double v) {
  return __longlong_as_double((long long)wave_join((unsigned long long)__double_as_longlong(v), [](auto a, auto b) {
    return (unsigned long long)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
  }));
}
// The wave's largest v.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t max_with_moved(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_with_moved<0x111, 0xF>(v);
  v = max_with_moved<0x112, 0xF>(v);
  v = max_with_moved<0x114, 0xF>(v);
  v = max_with_moved<0x118, 0xF>(v);
  v = max_with_moved<0x142, 0xA>(v);
  v = max_with_moved<0x143, 0xC>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
#endif

}  // namespace prom
