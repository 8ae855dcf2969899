// Rotary positions: channel pairs of queries and keys turned by position * frequency.
//
//   (a, b) -> m (a cos - b sin, b cos + a sin), the angle position * turns[i] revolutions,
// pairs (i, i + rotary / 2) or (2 i, 2 i + 1) of the first `rotary` channels of each head; the others are copied.
//
// A workgroup takes a row: its threads make the row's cosines and sines once, in LDS, and go over the heads with eight
// channels of each half (or eight neighbouring ones) a thread.  Angles are in binary64 and in revolutions, so that a
// far position loses nothing but whole turns; what is left of a turn is within 2^-24 in fp32, and sincospi is good to
// an ulp or two.  Bound by memory.
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

// kN channels of each of a pair's sides at once (kN = 1: any sizes).
template <typename T, bool kPairs, int kN>
__device__ __forceinline__ void turn_heads(const RopeArgs& a, const RopeTensor& x, size_t row, const float* cs) {
  const uint32_t half = a.rotary / 2;
  // Items of a head: kN pairs (halves) or kN / 2 (neighbours; one for kN = 1), then the channels that stay.
  const uint32_t per_item = kPairs && kN > 1 ? kN / 2 : kN;
  const uint32_t turned = half / per_item;
  const uint32_t stays = x.in != x.out ? (a.head_dim - a.rotary) / kN : 0;
  const uint32_t per_head = turned + stays, items = per_head * x.heads;
  const T* in = static_cast<const T*>(x.in) + row * x.in_stride;
  T* out = static_cast<T*>(x.out) + row * x.out_stride;
  for (uint32_t item = threadIdx.x; item < items; item += blockDim.x) {
    const uint32_t head = item / per_head, i = item - head * per_head;
    const T* from = in + (size_t)head * a.head_dim;
    T* to = out + (size_t)head * a.head_dim;
    if (i >= turned) {
      float v[kN];
      const uint32_t at = a.rotary + (i - turned) * kN;
      load(from + at, v);
      store(to + at, v);
      continue;
    }
    const uint32_t first = i * per_item;
    if constexpr (!kPairs) {
      float u[kN], v[kN];
      load(from + first, u);
      load(from + half + first, v);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float c = cs[2 * (first + j)], s = cs[2 * (first + j) + 1], p = u[j], q = v[j];
        u[j] = p * c - q * s;
        v[j] = q * c + p * s;
      }
      store(to + first, u);
      store(to + half + first, v);
    } else {
      constexpr int kBoth = kN > 1 ? kN : 2;
      float v[kBoth];
      load(from + 2 * first, v);
#pragma unroll
      for (int j = 0; j < kBoth; j += 2) {
        const float c = cs[2 * first + j], s = cs[2 * first + j + 1], p = v[j], q = v[j + 1];
        v[j] = p * c - q * s;
        v[j + 1] = q * c + p * s;
      }
      store(to + 2 * first, v);
    }
  }
}

template <typename T, bool kPairs, int kN>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
  __shared__ float cs[kRopeMaxDim];  // cosine and sine of each pair
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const double position = (double)a.positions[row];
    if (row != blockIdx.x) __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.rotary / 2; i += blockDim.x) {
      double t = position * a.turns[i];
      t -= rint(t);
      float s, c;
      sincospif(2.0f * (float)t, &s, &c);
      cs[2 * i] = c * a.magnitude;
      cs[2 * i + 1] = s * a.magnitude;
    }
    __syncthreads();
    if (a.q.in != nullptr) turn_heads<T, kPairs, kN>(a, a.q, row, cs);
    if (a.k.in != nullptr) turn_heads<T, kPairs, kN>(a, a.k, row, cs);
  }
}

template <typename T, bool kPairs>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)std::min<uint32_t>(a.rows, 1u << 20));
  // Eight channels at once where the sides and what stays are whole eights.
  if ((kPairs ? a.rotary : a.rotary / 2) % 8 == 0 && (a.head_dim - a.rotary) % 8 == 0)
    hipLaunchKernelGGL((rope_kernel<T, kPairs, 8>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, kPairs, 1>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool bf16, bool pairs, hipStream_t stream) {
  if (bf16) return pairs ? launch<uint16_t, true>(a, stream) : launch<uint16_t, false>(a, stream);
  return pairs ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace prom
