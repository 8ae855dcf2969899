// Groups of numbers held in 4 bits: the step and the codes of a group, and what they stand for.  Shared by the
// 4-bit cache (kv4_cache.hip) and the 4-bit weights (w4_matrix.hip).
//
// A group has a step s = max |x| / 6, rounded to fp32 and then up to six significant bits, and per number an
// E2M1 code: the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives to x / s.  x / s is the IEEE quotient
// and the conversion rounds halves to the even code: the codes are the definition's, bit for bit.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace prom {

typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kInfBits = 0x7F800000u;
constexpr uint32_t kNanParam = 0x7FC0u;  // the step of a group with an infinity or a NaN

__device__ __forceinline__ uint32_t max_bits(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return m;
}

// The largest of 4, 8 or 16 neighbouring lanes.
template <int kLanes>
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));  // the other of a pair
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));  // the other pair of four
  if constexpr (kLanes >= 8)
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));  // mirrored within eight
  if constexpr (kLanes >= 16)
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, true));  // mirrored within sixteen
  return m;
}

// The IEEE quotient x / d for d of at most six significant bits, r = 1 / d to within a few ulps: q = fl(x r)
// is a few ulps off, the remainder q d - x has few enough bits to be exact, and x / d lies 2^-7 ulps or
// more from where rounding changes, far more than the error of q - remainder r.  The sign of a zero is kept.
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = x * r;
  return __builtin_fmaf(-__builtin_fmaf(q, d, -x), r, q);
}

// Step (the upper half of an fp32) and codes of eight numbers of a group whose largest magnitude has the bits
// `m`.  Called by whole waves.
__device__ __forceinline__ uint32_t fp4_codes(const float (&v)[8], uint32_t m, uint32_t* param) {
  const float top = __uint_as_float(m);
  // In this range nothing under- or overflows on the way to a quotient that is not rounded to zero.
  const bool plain = (top >= 0x1p-80f && top <= 0x1p80f) || m == 0;
  const bool all_plain = __all(plain);
  const uint32_t t = __float_as_uint(all_plain ? quotient(top, 6.0f, 1.0f / 6.0f) : top / 6.0f);
  const float s = __uint_as_float((t + 0x3FFFFu) & 0xFFFC0000u);
  const bool finite = m < kInfBits;
  *param = finite ? __float_as_uint(s) >> 16 : kNanParam;
  const bool some = finite && s > 0.0f;
  const float d = some ? s : 1.0f;
  float y[8];
  if (all_plain) {
    const float r = __builtin_amdgcn_rcpf(d);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = quotient(v[j], d, r);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = v[j] / d;
  }
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[0], y[1], 1.0f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], 1.0f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[4], y[5], 1.0f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[6], y[7], 1.0f, 3);
  return some ? codes : 0u;
}

__device__ __forceinline__ void fp4_values(uint32_t codes, uint32_t param, float (&v)[8]) {
  const float s = __uint_as_float(param << 16);
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const floatx2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const floatx2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  v[0] = a.x * s, v[1] = a.y * s, v[2] = b.x * s, v[3] = b.y * s;
  v[4] = c.x * s, v[5] = c.y * s, v[6] = d.x * s, v[7] = d.y * s;
}

}  // namespace prom
