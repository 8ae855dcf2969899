// Rotary positions: channel pairs of queries and keys turned by position * frequency.
//
//   (a, b) -> m (a cos - b sin, b cos + a sin), the angle position * turns[i] revolutions,
// pairs (i, i + rotary / 2) or (2 i, 2 i + 1) of the first `rotary` channels of each head; the others are copied.
//
// A workgroup takes a row, or four: its threads make the rows' cosines and sines once, in LDS, and go over the heads with eight
// channels of each half (or eight neighbouring ones) a thread.  Angles, sines and cosines are in binary64 and in
// revolutions, so that a far position loses nothing but whole turns; they are rounded once to fp32 (a fraction of a turn and
// sincospif in fp32: 5.9e-8 of fp32 rows instead of 4.1e-8).  Bound by memory.
#include <algorithm>

#include "reactor_internal.h"

namespace prom {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int kN>
__device__ __forceinline__ void load(const float* p, float (&v)[kN]) {
  __builtin_memcpy(v, p, 4 * kN);
}
template <int kN>
__device__ __forceinline__ void load(const uint16_t* p, float (&v)[kN]) {
  uint16_t w[kN];
  __builtin_memcpy(w, p, 2 * kN);
#pragma unroll
  for (int j = 0; j < kN; ++j) v[j] = __uint_as_float((uint32_t)w[j] << 16);
}
template <int kN>
__device__ __forceinline__ void store(float* p, const float (&v)[kN]) {
  __builtin_memcpy(p, v, 4 * kN);
}
template <int kN>
__device__ __forceinline__ void store(uint16_t* p, const float (&v)[kN]) {
  __bf16 w[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) w[j] = (__bf16)v[j];
  __builtin_memcpy(p, w, 2 * kN);
}

// Cosine and sine of t revolutions, |t| <= 1/2, times m.  Within an eighth of the nearest quarter they are the power series of
// x = 2 pi t, |x| <= pi / 4, whose first terms left out are x^15 / 15! and x^16 / 16!, below 2^-45 and 2^-49.
__device__ __forceinline__ void turned(double t, double m, float* c, float* s) {
  const double quarter = rint(4.0 * t), x = 6.283185307179586 * __builtin_fma(-0.25, quarter, t), z = x * x;
  double sine = 1.0 / 6227020800.0, cosine = -1.0 / 87178291200.0;  // 1 / 13!, 1 / 14!
  sine = __builtin_fma(sine, z, -1.0 / 39916800.0), cosine = __builtin_fma(cosine, z, 1.0 / 479001600.0);
  sine = __builtin_fma(sine, z, 1.0 / 362880.0), cosine = __builtin_fma(cosine, z, -1.0 / 3628800.0);
  sine = __builtin_fma(sine, z, -1.0 / 5040.0), cosine = __builtin_fma(cosine, z, 1.0 / 40320.0);
  sine = __builtin_fma(sine, z, 1.0 / 120.0), cosine = __builtin_fma(cosine, z, -1.0 / 720.0);
  sine = __builtin_fma(sine, z, -1.0 / 6.0), cosine = __builtin_fma(cosine, z, 1.0 / 24.0);
  sine = x * __builtin_fma(sine, z, 1.0), cosine = __builtin_fma(__builtin_fma(cosine, z, -0.5), z, 1.0);
  const int q = (int)quarter;
  const double a = q & 1 ? -sine : cosine, b = q & 1 ? cosine : sine;  // a quarter turns (c, s) to (-s, c)
  *c = (float)(q & 2 ? -m * a : m * a);
  *s = (float)(q & 2 ? -m * b : m * b);
}

// kN channels of each of a pair's sides at once (kN = 1: any sizes), of row `r` of a workgroup's kRows, whose angles are
// cs[r][..].
template <typename T, bool kPairs, int kN, int kRows>
__device__ __forceinline__ void turn_heads(const RopeArgs& a, const RopeTensor& x, uint32_t row0, uint32_t rows,
                                           const float* cs) {
  const uint32_t half = a.rotary / 2;
  // Items of a head: kN pairs (halves) or kN / 2 (neighbours; one for kN = 1), then the channels that stay.
  const uint32_t per_item = kPairs && kN > 1 ? kN / 2 : kN;
  const uint32_t turned = half / per_item;
  const uint32_t stays = x.in != x.out ? (a.head_dim - a.rotary) / kN : 0;
  const uint32_t per_head = turned + stays, heads = x.heads * rows;
  // Item i of head `head` (of all rows'); 256 items further on is `skip` heads and `step` items.
  const uint32_t skip = 256 / per_head, step = 256 - skip * per_head;
  uint32_t head = threadIdx.x / per_head, i = threadIdx.x - head * per_head;
  uint32_t r = 0, of_row = head;  // its row, and its number within the row
  for (; head < heads; head += skip) {
    while (of_row >= x.heads) of_row -= x.heads, ++r;
    const T* from = static_cast<const T*>(x.in) + (size_t)(row0 + r) * x.in_stride + (size_t)of_row * a.head_dim;
    T* to = static_cast<T*>(x.out) + (size_t)(row0 + r) * x.out_stride + (size_t)of_row * a.head_dim;
    const float* angles = cs + r * a.rotary;
    if (i >= turned) {
      float v[kN];
      const uint32_t at = a.rotary + (i - turned) * kN;
      load(from + at, v);
      store(to + at, v);
    } else if constexpr (!kPairs) {
      const uint32_t first = i * per_item;
      float u[kN], v[kN];
      load(from + first, u);
      load(from + half + first, v);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float c = angles[2 * (first + j)], s = angles[2 * (first + j) + 1], p = u[j], q = v[j];
        u[j] = p * c - q * s;
        v[j] = q * c + p * s;
      }
      store(to + first, u);
      store(to + half + first, v);
    } else {
      constexpr int kBoth = kN > 1 ? kN : 2;
      const uint32_t first = i * per_item;
      float v[kBoth];
      load(from + 2 * first, v);
#pragma unroll
      for (int j = 0; j < kBoth; j += 2) {
        const float c = angles[2 * first + j], s = angles[2 * first + j + 1], p = v[j], q = v[j + 1];
        v[j] = p * c - q * s;
        v[j + 1] = q * c + p * s;
      }
      store(to + 2 * first, v);
    }
    of_row += skip;
    i += step;
    if (i >= per_head) i -= per_head, ++head, ++of_row;
  }
}

template <typename T, bool kPairs, int kN, int kRows>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
  extern __shared__ float cs[];  // [kRows][rotary]: cosine and sine of each pair
  const uint32_t half = a.rotary / 2, blocks = (a.rows + kRows - 1) / kRows;
  for (uint32_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const uint32_t row0 = block * kRows, rows = min(a.rows - row0, (uint32_t)kRows);
    if (block != blockIdx.x) __syncthreads();
    for (uint32_t at = threadIdx.x; at < rows * half; at += blockDim.x) {
      const uint32_t r = at / half, i = at - r * half;
      double t = (double)a.positions[row0 + r] * a.turns[i];
      t -= rint(t);
      turned(t, (double)a.magnitude, &cs[2 * at], &cs[2 * at + 1]);
    }
    __syncthreads();
    if (a.q.in != nullptr) turn_heads<T, kPairs, kN, kRows>(a, a.q, row0, rows, cs);
    if (a.k.in != nullptr) turn_heads<T, kPairs, kN, kRows>(a, a.k, row0, rows, cs);
  }
}

template <typename T, bool kPairs, int kN>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
  const unsigned one = a.rotary * sizeof(float);
#define ROPE(R)                                                                                                   \
  hipLaunchKernelGGL((rope_kernel<T, kPairs, kN, R>), dim3(std::min<unsigned>((a.rows + R - 1) / R, 1u << 20)),   \
                     dim3(256), R * one, stream, a)
  // Several rows a workgroup fill its last round of 256 items better (8191 rows of 32 + 8 heads of 128, half turned, bf16:
  // 37 us with one, 34 with four, 43 with eight); few rows keep all CUs busy one by one.
  if (a.rows < 4096)
    ROPE(1);
  else
    ROPE(4);
#undef ROPE
  return hipGetLastError();
}
template <typename T, bool kPairs>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
  // Eight channels at once where the sides and what stays are whole eights, else four, two or one (8191 rows of 40 heads,
  // 60 of 128 channels turned, one at once 84 us, 39 with four).
  const uint32_t whole = (kPairs ? a.rotary : a.rotary / 2) | (a.head_dim - a.rotary);
  if (whole % 8 == 0) return launch<T, kPairs, 8>(a, stream);
  if (whole % 4 == 0) return launch<T, kPairs, 4>(a, stream);
  if (whole % 2 == 0) return launch<T, kPairs, 2>(a, stream);
  return launch<T, kPairs, 1>(a, stream);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool bf16, bool pairs, hipStream_t stream) {
  if (bf16) return pairs ? launch<uint16_t, true>(a, stream) : launch<uint16_t, false>(a, stream);
  return pairs ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace prom
