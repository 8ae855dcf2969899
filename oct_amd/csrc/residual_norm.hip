// The residual sum between two blocks with the norms before and after it:
//   h' = h + residual_scale * g * norm(y; post),  out = norm(h'; pre) * (1 + scale) + shift,
// norm(x; w) = x / sqrt(mean(x^2) + eps) * w.
//
// A row is read once into registers and both norms are taken from there: bound by memory, and for the few rows of a decode
// step by the chain of two sums over a workgroup.  Squares are summed in binary64, which holds those of every fp32 number.
// The second norm is that of h' before it is rounded to a bf16 row.  A workgroup takes neighbouring rows and keeps what
// they share, the weights and vectors joined to a factor of y, a factor of h' and a summand, in registers (read again for
// each row, 4224 rows of 3840 in bf16 took 53 us); the next row is loaded meanwhile.  Those rows take 31 us, 130 MB at 4.2
// TB/s; a large copy runs at 5.1.
#include <algorithm>

#include "reactor_internal.h"
#include "wave_ops.h"

namespace prom {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight values of a row as they lie in memory.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
  float v[8];
  __device__ __forceinline__ void get(float (&to)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j] = v[j];
  }
};
template <>
struct Raw<uint16_t> {
  u32x4 w;
  __device__ __forceinline__ void get(float (&to)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      to[2 * j] = __uint_as_float(w[j] << 16);
      to[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
};
// From p (any alignment of T), zeros from the left-th on; kWhole: all eight are there.
template <bool kWhole>
__device__ __forceinline__ Raw<float> load8(const float* p, int left) {
  Raw<float> r;
  if (kWhole || left >= 8) {
    __builtin_memcpy(r.v, p, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = j < left ? p[j] : 0.0f;
  }
  return r;
}
template <bool kWhole>
__device__ __forceinline__ Raw<uint16_t> load8(const uint16_t* p, int left) {
  Raw<uint16_t> r;
  if (kWhole || left >= 8) {
    __builtin_memcpy(&r.w, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r.w[j] = (2 * j < left ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < left ? (uint32_t)p[2 * j + 1] << 16 : 0u);
  }
  return r;
}
template <bool kWhole>
__device__ __forceinline__ void store8(float* p, int left, const float (&v)[8]) {
  if (kWhole || left >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = v[j];
  }
}
template <bool kWhole>
__device__ __forceinline__ void store8(uint16_t* p, int left, const float (&v)[8]) {
  __bf16 w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = (__bf16)v[j];
  if (kWhole || left >= 8) {
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
  v = wave_sum(v);
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w];
  }
  return v;
}
// 1 / sqrt(mean + eps) as a product: past fp32's range, or where it would be among its subnormal numbers (rows below 2^-100,
// above 2^100), `scale` is the power of two that keeps x scale and `rest` within it.
struct Inverse {
  float scale, rest;
  __device__ __forceinline__ float of(float x) const { return x * scale * rest; }
};
// Of a sum of squares, over = 1 / width: the instruction's value is within 2^-23 or so, a step of
// Newton's makes it 2^-45 (a division and a root in binary64 were a third of the kernel's time).  Where the step has no
// value the root's is that of 0 or infinity, and stands.
__device__ __forceinline__ Inverse inverse_size(double sum, double over, float eps) {
  const double x = __builtin_fma(sum, over, (double)eps), q = __builtin_amdgcn_rsq(x), e = __builtin_fma(-x * q, q, 1.0);
  const double r = e == e ? __builtin_fma(0.5 * q, e, q) : q;
  if (r > 0x1p100) return Inverse{0x1p64f, (float)(r * 0x1p-64)};
  if (r < 0x1p-100) return Inverse{0x1p-64f, (float)(r * 0x1p64)};
  return Inverse{1.0f, (float)r};
}

// The squares' sum of eight values of which there are `left`, if any; what lies behind them is zero where it is not a repeat.
__device__ __forceinline__ double squares(const float (&v)[8], int left) {
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)v[j], (double)v[j], sum);
  return left > 0 ? sum : 0.0;
}

// kWaves waves a row (with one, four rows a workgroup at once), kChunks groups of eight values a lane.  A workgroup takes rows
// blockIdx.x * share ..  kWhole: the width is whole eights; the lanes behind it load the last eight and leave them out, so that
// nothing branches between a load and its use (there the compiler waited for the row's stores too: 42 us instead of 31).
template <typename T, int kWaves, int kChunks, bool kWhole>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void residual_norm_kernel(const ResidualNormArgs a,
                                                                                         uint32_t share) {
  constexpr int kRows = kWaves == 1 ? 4 : 1, kLanes = 64 * kWaves;
  __shared__ double part[2][2][kWaves];
  const int lane = kWaves == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  const int width = (int)a.width;
  int at[kChunks], left[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    at[i] = 8 * (lane + kLanes * i);
    left[i] = max(width - at[i], 0);
    at[i] = min(at[i], kWhole ? width - 8 : width);
  }
  uint32_t row = blockIdx.x * share + (kWaves == 1 ? threadIdx.x >> 6 : 0);
  const uint32_t end = min(a.rows, (blockIdx.x + 1) * share);
  if (row >= end) return;  // with several waves all agree
  Raw<T> h_next[kChunks], y_next[kChunks];
  const auto fetch = [&](uint32_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      h_next[i] = load8<kWhole>(static_cast<const T*>(a.h) + (size_t)r * a.h_stride + at[i], left[i]);
      if (a.y != nullptr) y_next[i] = load8<kWhole>(static_cast<const T*>(a.y) + (size_t)r * a.y_stride + at[i], left[i]);
    }
  };
  // What h' takes of y / its size, and what out takes of h' / its size, for chunk i of a row with vector number `vector`.
  const auto of_y = [&](uint32_t vector, int i, float (&f)[8]) __attribute__((always_inline)) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = a.residual_scale;
    if (a.post != nullptr) {
      load8<kWhole>(a.post + at[i], left[i]).get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= a.weight_offset + v[j];
    }
    if (a.gate != nullptr) {
      load8<kWhole>(static_cast<const T*>(a.gate) + (size_t)vector * a.vector_stride + at[i], left[i]).get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= a.gate_tanh ? tanhf(v[j]) : v[j];
    }
  };
  const auto of_h = [&](uint32_t vector, int i, float (&f)[8], float (&add)[8]) __attribute__((always_inline)) {
    const size_t from = (size_t)vector * a.vector_stride + at[i];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 1.0f, add[j] = 0.0f;
    if (a.pre != nullptr) {
      load8<kWhole>(a.pre + at[i], left[i]).get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = a.weight_offset + v[j];
    }
    if (a.scale != nullptr) {
      load8<kWhole>(static_cast<const T*>(a.scale) + from, left[i]).get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= 1.0f + v[j];
    }
    if (a.shift != nullptr) load8<kWhole>(static_cast<const T*>(a.shift) + from, left[i]).get(add);
  };
  // Rows of several chunks a lane have no registers for the next row (900 rows of 16384 in bf16 28 us, with it 32), those of
  // four none for these either (500 rows of 32768 70 us, with them 117).
  constexpr bool kKeeps = kChunks <= 2, kAhead = kChunks == 1;
  if constexpr (kAhead) fetch(row);
  constexpr int kKept = kKeeps ? kChunks : 1, kStays = kKeeps ? 1 : 0;
  float fy[kKept][8], fh[kKept][8], add[kKept][8];
  uint32_t vector = 0xFFFFFFFFu;  // the vectors that the factors are of
  int turn = 0;
  for (; row < end; row += kRows) {
    if constexpr (!kAhead) fetch(row);
    if (row / a.rows_per_vector != vector) {
      vector = row / a.rows_per_vector;
      if constexpr (kKeeps)
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          of_y(vector, i, fy[i]);
          of_h(vector, i, fh[i], add[i]);
        }
    }
    float h[kChunks][8], y[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      h_next[i].get(h[i]);
      if (a.y != nullptr) y_next[i].get(y[i]);
    }
    if constexpr (kAhead)
      if (row + kRows < end) fetch(row + kRows);
    const uint32_t now = row;
    if (a.y != nullptr) {
      Inverse r{1.0f, 1.0f};
      if (a.post != nullptr) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) sum += squares(y[i], left[i]);
        r = inverse_size(row_sum<kWaves>(sum, part[0][turn]), a.over_width, a.eps);
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (!kKeeps) of_y(vector, i, fy[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = __builtin_fmaf(r.of(y[i][j]), fy[kStays * i][j], h[i][j]);
      }
    }
    if (a.h_out != nullptr) {
      T* to = static_cast<T*>(a.h_out) + (size_t)now * a.h_out_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        if (left[i] > 0) store8<kWhole>(to + at[i], left[i], h[i]);
    }
    if (a.out != nullptr) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) sum += squares(h[i], left[i]);
      const Inverse r = inverse_size(row_sum<kWaves>(sum, part[1][turn]), a.over_width, a.eps);
      T* to = static_cast<T*>(a.out) + (size_t)now * a.out_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if constexpr (!kKeeps) of_h(vector, i, fh[0], add[0]);
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j] = r.of(h[i][j]) * fh[kStays * i][j];
          if (a.shift != nullptr) o[j] += add[kStays * i][j];
        }
        if (left[i] > 0) store8<kWhole>(to + at[i], left[i], o);
      }
    }
    // Parts are written again two rows on: a barrier of the next row lies between, if rows have any.
    turn ^= 1;
  }
}

template <typename T, bool kWhole>
hipError_t launch(const ResidualNormArgs& a, hipStream_t stream) {
#define ROWS(W, C, WGS)                                                                              \
  {                                                                                                  \
    const uint32_t at_once = W == 1 ? 4u : 1u, groups = (a.rows + at_once - 1) / at_once;            \
    const uint32_t share = (groups + WGS - 1) / WGS * at_once;                                       \
    hipLaunchKernelGGL((residual_norm_kernel<T, W, C, kWhole>), dim3((a.rows + share - 1) / share),  \
                       dim3(W == 1 ? 256 : 64 * W), 0, stream, a, share);                            \
  }
  // As many waves a row as hold it in eight values a lane (with half the waves and 16 values: 4224 rows of 3840 35 us
  // instead of 31, 1483 of 8192 36 instead of 26), and about as many workgroups as run at once: with twice as many their
  // first rows' latency and the joining of the vectors came twice (34 us).
  if (a.width <= 512)
    ROWS(1, 1, 1024)
  else if (a.width <= 1024)
    ROWS(2, 1, 2048)
  else if (a.width <= 2048)
    ROWS(4, 1, 1024)
  else if (a.width <= 4096)
    ROWS(8, 1, 512)
  else if (a.width <= 8192)
    ROWS(16, 1, 256)
  else if (a.width <= 16384)
    ROWS(16, 2, 256)
  else
    ROWS(16, 4, 256)
#undef ROWS
  return hipGetLastError();
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormArgs& a, bool bf16, hipStream_t stream) {
  if (a.width % 8 == 0) return bf16 ? launch<uint16_t, true>(a, stream) : launch<float, true>(a, stream);
  return bf16 ? launch<uint16_t, false>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace prom
