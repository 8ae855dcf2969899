// The residual sum between two blocks with the norms before and after it:
//   h' = h + residual_scale * g * norm(y; post),  out = norm(h'; pre) * (1 + scale) + shift,
// norm(x; w) = x / sqrt(mean(x^2) + eps) * w.
//
// A row is read once into registers and both norms are taken from there: bound by memory, and for the few rows of
// a decode step by the chain of two sums over a workgroup.  Squares are summed in binary64, which holds those of every
// fp32 number.  The second norm is that of h' before it is rounded to a bf16 row.
#include <algorithm>

#include "reactor_internal.h"

namespace prom {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight values from p (any alignment of T), zeros from the left-th on.
__device__ __forceinline__ void load8(const float* p, int left, float (&v)[8]) {
  if (left >= 8) {
    __builtin_memcpy(v, p, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
__device__ __forceinline__ void load8(const uint16_t* p, int left, float (&v)[8]) {
  if (left >= 8) {
    u32x4 w;
    __builtin_memcpy(&w, p, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? __uint_as_float((uint32_t)p[j] << 16) : 0.0f;
  }
}
__device__ __forceinline__ void store8(float* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = v[j];
  }
}
__device__ __forceinline__ void store8(uint16_t* p, int left, const float (&v)[8]) {
  __bf16 w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = (__bf16)v[j];
  if (left >= 8) {
    __builtin_memcpy(p, w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = __builtin_bit_cast(uint16_t, w[j]);
  }
}

// The sum over a row's lanes, in every lane.
template <int kWaves>
__device__ __forceinline__ double row_sum(double v, double (&part)[kWaves]) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w];
  }
  return v;
}

template <int kChunks>
__device__ __forceinline__ double squares(const float (&v)[kChunks][8]) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fma((double)v[i][j], (double)v[i][j], s);
  return s;
}

// kWaves waves a row (with one, four rows a workgroup), kChunks groups of eight values a lane.
template <typename T, int kWaves, int kChunks>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void residual_norm_kernel(const ResidualNormArgs a) {
  constexpr int kRows = kWaves == 1 ? 4 : 1, kLanes = 64 * kWaves;
  __shared__ double part[2][kWaves];
  const int lane = kWaves == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  const int width = (int)a.width;
  for (size_t row = (size_t)blockIdx.x * kRows + (kWaves == 1 ? threadIdx.x >> 6 : 0); row < a.rows;
       row += (size_t)gridDim.x * kRows) {
    const T* h_row = static_cast<const T*>(a.h) + row * a.h_stride;
    float h[kChunks][8], y[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = 8 * (lane + kLanes * i);
      load8(h_row + min(at, width), width - at, h[i]);
    }
    const size_t vector = (size_t)(row / a.rows_per_vector) * a.vector_stride;
    if (a.y != nullptr) {
      const T* y_row = static_cast<const T*>(a.y) + row * a.y_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int at = 8 * (lane + kLanes * i);
        load8(y_row + min(at, width), width - at, y[i]);
      }
      float r = a.residual_scale;
      if (a.post != nullptr) r *= (float)(1.0 / sqrt(row_sum<kWaves>(squares(y), part[0]) / width + (double)a.eps));
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int at = 8 * (lane + kLanes * i), left = width - at;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = r;
        if (a.post != nullptr) {
          float w[8];
          load8(a.post + min(at, width), left, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= a.weight_offset + w[j];
        }
        if (a.gate != nullptr) {
          float g[8];
          load8(static_cast<const T*>(a.gate) + vector + min(at, width), left, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= a.gate_tanh ? tanhf(g[j]) : g[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = __builtin_fmaf(y[i][j], f[j], h[i][j]);
      }
    }
    if (a.h_out != nullptr) {
      T* to = static_cast<T*>(a.h_out) + row * a.h_out_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int at = 8 * (lane + kLanes * i);
        if (at < width) store8(to + at, width - at, h[i]);
      }
    }
    if (a.out != nullptr) {
      T* to = static_cast<T*>(a.out) + row * a.out_stride;
      const float r = (float)(1.0 / sqrt(row_sum<kWaves>(squares(h), part[1]) / width + (double)a.eps));
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int at = 8 * (lane + kLanes * i), left = width - at;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = h[i][j] * r;
        if (a.pre != nullptr) {
          float w[8];
          load8(a.pre + min(at, width), left, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= a.weight_offset + w[j];
        }
        if (a.scale != nullptr) {
          float s[8];
          load8(static_cast<const T*>(a.scale) + vector + min(at, width), left, s);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= 1.0f + s[j];
        }
        if (a.shift != nullptr) {
          float s[8];
          load8(static_cast<const T*>(a.shift) + vector + min(at, width), left, s);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] += s[j];
        }
        if (left > 0) store8(to + at, left, f);
      }
    }
    if constexpr (kWaves > 1) __syncthreads();  // the parts are read
  }
}

template <typename T>
hipError_t launch(const ResidualNormArgs& a, hipStream_t stream) {
  const unsigned one = (unsigned)std::min<uint64_t>(a.rows, 1u << 20);
  const unsigned four = (unsigned)std::min<uint64_t>((a.rows + 3ull) / 4, 1u << 20);
#define ROWS(W, C, grid, block) \
  hipLaunchKernelGGL((residual_norm_kernel<T, W, C>), dim3(grid), dim3(block), 0, stream, a)
  if (a.width <= 512)
    ROWS(1, 1, four, 256);
  else if (a.width <= 2048)
    ROWS(4, 1, one, 256);
  else if (a.width <= 4096)
    ROWS(8, 1, one, 512);
  else if (a.width <= 8192)
    ROWS(8, 2, one, 512);
  else if (a.width <= 16384)
    ROWS(16, 2, one, 1024);
  else
    ROWS(16, 4, one, 1024);
#undef ROWS
  return hipGetLastError();
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<uint16_t>(a, stream) : launch<float>(a, stream);
}

}  // namespace prom
