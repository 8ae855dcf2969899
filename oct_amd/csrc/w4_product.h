// Products of a few rows with 4-bit weights, the part that gemm_w4.hip and moe_w4.hip share: one wave's sums over
// a range of K.
//
// D = X W^T by v_mfma_f32_16x16x32_bf16 with the rows of x as A and the weights' codes, exact in bf16, as B: lane l
// then holds columns l % 16 and rows 4 (l / 16) .. + 3 of the sums, so that a column's step is one value a lane.  A
// group's sum is multiplied by its step (one fused multiply-add for each of its four rows) rather than each weight:
// 512 weights of a step are 8 a lane.  bf16 rows enter as they are; fp32 rows as three bf16 terms, exact (8 + 8 + 8
// significant bits).
#pragma once

#include "w4_tiles.h"

namespace prom {

// Rows of x as one lane sees them: `p` is its row's first element (any aligned address where the lane has no row).
struct W4RowsBf16 {
  static constexpr int kTerms = 1;
  typedef uint16_t Element;
  struct Raw {
    u32x4 v;
  };
  const uint16_t* p;
  bool live;
  // Eight columns from `at`; zeros for a lane without a row and, where kTail, from column k on.
  template <bool kTail>
  __device__ __forceinline__ Raw fetch(int at, int k) const {
    Raw r{u32x4{0u, 0u, 0u, 0u}};
    if (!live) return r;
    if (!kTail || at + 8 <= k) {
      __builtin_memcpy(&r.v, p + at, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < k) r.v[j >> 1] |= (uint32_t)p[at + j] << (16 * (j & 1));
    }
    return r;
  }
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[1]) { x[0] = __builtin_bit_cast(bf16x8, r.v); }
};

struct W4RowsF32 {
  static constexpr int kTerms = 3;
  typedef float Element;
  struct Raw {
    float v[8];
  };
  const float* p;
  bool live;
  template <bool kTail>
  __device__ __forceinline__ Raw fetch(int at, int k) const {
    Raw r{};
    if (!live) return r;
    if (!kTail || at + 8 <= k) {
      __builtin_memcpy(r.v, p + at, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < k) r.v[j] = p[at + j];
    }
    return r;
  }
  // x = x[0] + x[1] + x[2], each the upper half of what the ones before leave.  An infinity is its first term.
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[3]) {
    u32x4 t[3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t part[2][3];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v = r.v[2 * j + i];
        part[i][0] = __float_as_uint(v);
        const float high = __uint_as_float(part[i][0] & 0xFFFF0000u);
        const float rest = __builtin_fabsf(v) == __builtin_inff() ? 0.0f : v - high;
        part[i][1] = __float_as_uint(rest);
        part[i][2] = __float_as_uint(rest - __uint_as_float(part[i][1] & 0xFFFF0000u));
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) t[i][j] = __builtin_amdgcn_perm(part[1][i], part[0][i], 0x07060302u);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) x[i] = __builtin_bit_cast(bf16x8, t[i]);
  }
};

// A lane's steps of one tile, its column's kSteps = 128 / group.
template <int kSteps>
struct W4Steps {
  uint32_t v[kSteps > 1 ? kSteps / 2 : 1];
  __device__ __forceinline__ void fetch(const uint16_t* p) {
    if constexpr (kSteps == 1)
      v[0] = *p;
    else
      __builtin_memcpy(v, p, 2 * kSteps);
  }
  __device__ __forceinline__ float operator[](int i) const {
    return __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
  }
};

// kNT tiles of columns (codes and steps as w4_codes and w4_steps give them) by kMT times sixteen rows: adds tiles kt,
// kt + stride, ... (kDepth of them, which all exist) of K.  The codes of all are asked for before the first is used.
template <int kSteps, int kNT, int kMT, int kDepth, bool kTail, typename X>
__device__ __forceinline__ void w4_add_tiles(const u32x4* const (&codes)[kNT], const uint16_t* const (&steps)[kNT],
                                             const X (&x)[kMT], int live_mt, int kt, int stride, int k,
                                             floatx4 (&acc)[kMT][kNT]) {
  const int lane = (int)threadIdx.x & 63;
  u32x4 c[kDepth][kNT];
  W4Steps<kSteps> s[kDepth][kNT];
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      const int at = kt + d * stride;
      c[d][i] = codes[i][(size_t)at * 64 + lane];
      s[d][i].fetch(steps[i] + ((size_t)at * 16 + (lane & 15)) * kSteps);
    }
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    const int first = (kt + d * stride) * kW4TileK + 8 * (lane >> 4);
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      if (kMT > 1 && m >= live_mt) break;
      typename X::Raw raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) raw[u] = x[m].template fetch<kTail>(first + 32 * u, k);
#pragma unroll
      for (int g = 0; g < kSteps; ++g) {
        floatx4 sum[kNT];
#pragma unroll
        for (int i = 0; i < kNT; ++i) sum[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = g * (4 / kSteps); u < (g + 1) * (4 / kSteps); ++u) {
          bf16x8 xs[X::kTerms];
          X::terms(raw[u], xs);
#pragma unroll
          for (int i = 0; i < kNT; ++i) {
            const bf16x8 w = w4_numbers(c[d][i][u]);
#pragma unroll
            for (int t = X::kTerms - 1; t >= 0; --t)
              sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xs[t], w, sum[i], 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < kNT; ++i) acc[m][i] += sum[i] * s[d][i][g];
      }
    }
  }
}

// Tiles kt, kt + stride, ... below `end` of K, whose last tile is `k` columns' last.
template <int kSteps, int kNT, int kMT, int kDepth, typename X>
__device__ __forceinline__ void w4_accumulate(const u32x4* const (&codes)[kNT], const uint16_t* const (&steps)[kNT],
                                              const X (&x)[kMT], int live_mt, int kt, int end, int stride, int k,
                                              floatx4 (&acc)[kMT][kNT]) {
  const int whole = min(end, k / kW4TileK);
  for (; kt + (kDepth - 1) * stride < whole; kt += kDepth * stride)
    w4_add_tiles<kSteps, kNT, kMT, kDepth, false>(codes, steps, x, live_mt, kt, stride, k, acc);
  if (kDepth > 2 && kt + stride < whole) {
    w4_add_tiles<kSteps, kNT, kMT, 2, false>(codes, steps, x, live_mt, kt, stride, k, acc);
    kt += 2 * stride;
  }
  for (; kt < whole; kt += stride)
    w4_add_tiles<kSteps, kNT, kMT, 1, false>(codes, steps, x, live_mt, kt, stride, k, acc);
  if (kt < end) w4_add_tiles<kSteps, kNT, kMT, 1, true>(codes, steps, x, live_mt, kt, stride, k, acc);
}

}  // namespace prom
