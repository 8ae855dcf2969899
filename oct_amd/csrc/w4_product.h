// Products of a few rows with 4-bit weights, the part that gemm_w4.hip and moe_w4.hip share: one wave's sums over
// a range of K.
//
// D = X W^T by v_mfma_f32_16x16x32_bf16 with the rows of x as A and the weights' codes, exact in bf16, as B: lane l
// then holds columns l % 16 and rows 4 (l / 16) .. + 3 of the sums, so that a column's step is one value a lane.  A
// group's sum is multiplied by its step (one fused multiply-add for each of its four rows) rather than each weight:
// 512 weights of a step are 8 a lane.  bf16 rows enter as they are; fp32 rows as three bf16 terms, exact (8 + 8 + 8
// significant bits) but for what an element has below 2^-133, bf16's smallest number.
//
// A tile travels from memory to registers while the one before is used, x with it.  Loads are never skipped: lanes
// without a row load the last row (its sums are not used), and behind the last tile that one is loaded again, so that
// the compiler's waits count loads exactly.
#pragma once

#include "w4_tiles.h"

namespace prom {

// How the end of K meets a tile's 128 columns.
enum W4Edge {
  kEdgeNone,   // k is a multiple of 128
  kEdgeShift,  // the last tile's columns past k are cut off; k >= 8
  kEdgeOdd,    // the same for bf16 rows that do not all lie on words' borders
  kEdgeShort,  // k < 8
};

// The edge of products with rows of x `stride` elements of T apart, the first at p.
template <typename T>
W4Edge w4_edge(const void* p, size_t stride, int k) {
  if (k < 8) return kEdgeShort;
  if (((uintptr_t)p | stride * sizeof(T)) % 4 != 0) return kEdgeOdd;
  return k % kW4TileK == 0 ? kEdgeNone : kEdgeShift;
}

// Eight 16-bit values less the first d (0..8), zeros from behind.
__device__ __forceinline__ u32x4 w4_drop(u32x4 v, int d) {
  unsigned long long low = (unsigned long long)v[1] << 32 | v[0], high = (unsigned long long)v[3] << 32 | v[2];
  if (d >= 4) low = high, high = 0, d -= 4;
  if (d >= 4) low = 0, d = 0;
  if (d > 0) low = low >> (16 * d) | high << (64 - 16 * d), high >>= 16 * d;
  return u32x4{(uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32)};
}

// Rows of x as one lane sees them: `p` is its row's first element.  fetch loads the eight columns from `at`, or where
// they reach past k those that end there (kEdgeShift, kEdgeOdd: their terms are shifted before they are used).
struct W4RowsBf16 {
  static constexpr int kTerms = 1;
  typedef uint16_t Element;
  struct Raw {
    u32x4 v;
    uint32_t behind, shift;  // kEdgeOdd: the word behind v, and where in v's first word the first column is
  };
  const uint16_t* p;
  template <W4Edge kEdge>
  __device__ __forceinline__ Raw fetch(int at, int k) const {
    Raw r{};
    if constexpr (kEdge == kEdgeShort) {
      for (int j = 0; j < 8; ++j)
        if (at + j < k) r.v[j >> 1] |= (uint32_t)p[at + j] << (16 * (j & 1));
    } else if constexpr (kEdge == kEdgeOdd) {
      // Whole words, each of which holds one of the columns or two (33 rows of 3001x1999 7.7 us; with loads off words'
      // borders 10.9; on them 6.1, but 7.7 this way).
      const char* from = reinterpret_cast<const char*>(p + min(at, k - 8));
      const uint32_t odd = (uint32_t)(uintptr_t)from & 2u;
      __builtin_memcpy(&r.v, __builtin_assume_aligned(from - odd, 4), 16);
      __builtin_memcpy(&r.behind, __builtin_assume_aligned(from + 12 + odd, 4), 4);
      r.shift = 8 * odd;
    } else {
      __builtin_memcpy(&r.v, p + (kEdge == kEdgeShift ? min(at, k - 8) : at), 16);
    }
    return r;
  }
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[1]) {
    const u32x4 v{__builtin_amdgcn_alignbit(r.v[1], r.v[0], r.shift), __builtin_amdgcn_alignbit(r.v[2], r.v[1], r.shift),
                  __builtin_amdgcn_alignbit(r.v[3], r.v[2], r.shift), __builtin_amdgcn_alignbit(r.behind, r.v[3], r.shift)};
    x[0] = __builtin_bit_cast(bf16x8, v);
  }
};

// Eight fp32 values as three bf16 terms each, the upper half of what the ones before leave.  An infinity is its first
// term.
__device__ __forceinline__ void w4_split(const float (&v)[8], u32x4 (&t)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t part[2][3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = v[2 * j + i];
      part[i][0] = __float_as_uint(x);
      const float high = __uint_as_float(part[i][0] & 0xFFFF0000u);
      const float rest = __builtin_fabsf(x) == __builtin_inff() ? 0.0f : x - high;
      part[i][1] = __float_as_uint(rest);
      part[i][2] = __float_as_uint(rest - __uint_as_float(part[i][1] & 0xFFFF0000u));
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) t[i][j] = __builtin_amdgcn_perm(part[1][i], part[0][i], 0x07060302u);
  }
}

struct W4RowsF32 {
  static constexpr int kTerms = 3;
  typedef float Element;
  struct Raw {
    float v[8];
  };
  const float* p;
  template <W4Edge kEdge>
  __device__ __forceinline__ Raw fetch(int at, int k) const {
    Raw r{};
    if constexpr (kEdge == kEdgeShort) {
      for (int j = 0; j < 8; ++j)
        if (at + j < k) r.v[j] = p[at + j];
    } else {
      __builtin_memcpy(r.v, p + (kEdge == kEdgeShift ? min(at, k - 8) : at), 32);
    }
    return r;
  }
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[3]) {
    u32x4 t[3];
    w4_split(r.v, t);
#pragma unroll
    for (int i = 0; i < 3; ++i) x[i] = __builtin_bit_cast(bf16x8, t[i]);
  }
};

// Rows that lie as bf16 terms in planes of 128-column tiles: memory or LDS, zeros behind the last column.
template <int kT>
struct W4RowsTerms {
  static constexpr int kTerms = kT;
  typedef uint16_t Element;
  struct Raw {
    u32x4 v[kT];
  };
  const uint16_t* p;
  size_t plane;
  template <W4Edge>
  __device__ __forceinline__ Raw fetch(int at, int) const {
    Raw r;
#pragma unroll
    for (int t = 0; t < kT; ++t) r.v[t] = *reinterpret_cast<const u32x4*>(p + t * plane + at);
    return r;
  }
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[kT]) {
#pragma unroll
    for (int t = 0; t < kT; ++t) x[t] = __builtin_bit_cast(bf16x8, r.v[t]);
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

// One tile of K, 16 kNT columns.
template <int kSteps, int kNT>
struct W4Tile {
  u32x4 c[kNT];
  W4Steps<kSteps> s[kNT];
  __device__ __forceinline__ void fetch(const u32x4* const (&codes)[kNT], const uint16_t* const (&steps)[kNT], int kt) {
    const int lane = (int)threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      c[i] = codes[i][(size_t)kt * 64 + lane];
      s[i].fetch(steps[i] + ((size_t)kt * 16 + (lane & 15)) * kSteps);
    }
  }
};

template <typename X, int kMT>
struct W4XTile {
  typename X::Raw r[kMT][4];
  template <W4Edge kEdge>
  __device__ __forceinline__ void fetch(const X (&x)[kMT], int kt, int k) {
    const int first = kt * kW4TileK + 8 * (((int)threadIdx.x & 63) >> 4);
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int u = 0; u < 4; ++u) r[m][u] = x[m].template fetch<kEdge>(first + 32 * u, k);
  }
};

// Tile kt; the last one's columns from k on are cut off.
template <int kSteps, int kNT, int kMT, W4Edge kEdge, typename X>
__device__ __forceinline__ void w4_add_tile(const W4Tile<kSteps, kNT>& w, const W4XTile<X, kMT>& x, int kt, int k,
                                            floatx4 (&acc)[kMT][kNT]) {
  const bool tail = (kEdge == kEdgeShift || kEdge == kEdgeOdd) && kt == k / kW4TileK;
#pragma unroll
  for (int g = 0; g < kSteps; ++g) {
    floatx4 sum[kMT][kNT];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int i = 0; i < kNT; ++i) sum[m][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = g * (4 / kSteps); u < (g + 1) * (4 / kSteps); ++u) {
      bf16x8 b[kNT];
#pragma unroll
      for (int i = 0; i < kNT; ++i) b[i] = w4_numbers(w.c[i][u]);
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        bf16x8 a[X::kTerms];
        X::terms(x.r[m][u], a);
        // The terms are shifted, not the fp32 values before the split: of that clang 22 made code that writes an element's
        // rest over the element before its upper half, the first term, is taken (groups of 128: seven of eight columns of a
        // tile's last step lost it).  The tests hold each column of a tile with all its bits.
        if (tail) {
          const int at = kt * kW4TileK + 32 * u + 8 * (((int)threadIdx.x & 63) >> 4);
          const int d = min(max(at + 8 - k, 0), 8);
#pragma unroll
          for (int t = 0; t < X::kTerms; ++t) a[t] = __builtin_bit_cast(bf16x8, w4_drop(__builtin_bit_cast(u32x4, a[t]), d));
        }
#pragma unroll
        for (int t = X::kTerms - 1; t >= 0; --t)
#pragma unroll
          for (int i = 0; i < kNT; ++i)
            sum[m][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t], b[i], sum[m][i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int i = 0; i < kNT; ++i) acc[m][i] += sum[m][i] * w.s[i][g];
  }
}

// Adds tiles kt, kt + stride, ... below `end` of K: kNT tiles of columns (codes and steps as w4_codes and w4_steps
// give them) by 16 kMT rows.  `first` is tile kt, asked for by the caller as soon as it knows its weights.
template <int kSteps, int kNT, int kMT, W4Edge kEdge, typename X>
__device__ __forceinline__ void w4_accumulate(const u32x4* const (&codes)[kNT], const uint16_t* const (&steps)[kNT],
                                              const W4Tile<kSteps, kNT>& first, const X (&x)[kMT], int kt, int end,
                                              int stride, int k, floatx4 (&acc)[kMT][kNT]) {
  if (kt >= end) return;
  const int last = kt + (end - 1 - kt) / stride * stride;
  W4Tile<kSteps, kNT> w[2];
  W4XTile<X, kMT> xs[2];
  w[0] = first;
  xs[0].template fetch<kEdge>(x, kt, k);
  const auto step = [&](int now) __attribute__((always_inline)) {
    const int next = min(kt + stride, last);
    w[now ^ 1].fetch(codes, steps, next);
    xs[now ^ 1].template fetch<kEdge>(x, next, k);
    asm volatile("" ::: "memory");  // the loads above stay above: the compiler would move them to their use
    w4_add_tile<kSteps, kNT, kMT, kEdge>(w[now], xs[now], kt, k, acc);
    const bool more = kt != last;
    kt += stride;
    return more;
  };
  while (step(0) && step(1)) {
  }
}

}  // namespace prom
