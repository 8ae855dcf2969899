// Rows quantised to 8-bit integers: q = rint(x / s) within -127..127, s = max |x| / 127, a row's
// own scale (the operand of the int8 product, gemm_int8.hip).
//
// Bound by memory: a row is read once into registers, reduced, and written as
// bytes.  The largest magnitude is the largest of the absolute values' bit
// patterns (an integer maximum, which also carries infinities and NaNs past
// every finite value).  x / s is the IEEE quotient, so that q is the same on
// every device that follows the definition.  4224 rows of 10240 in bf16: 25.8 us,
// 5.0 TB/s (with a division for each quotient 29); one row of 2048: a launch, 4.9.
#include "reactor_internal.h"

namespace prom {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kInfBits = 0x7F800000u;

// Eight values from p (any alignment of T), zeros from the left-th on.
__device__ __forceinline__ void load8(const float* p, long long left, float (&v)[8]) {
  if (left >= 8) {
    __builtin_memcpy(v, p, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
__device__ __forceinline__ void load8(const uint16_t* p, long long left, float (&v)[8]) {
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

__device__ __forceinline__ uint32_t max_bits(const float (&v)[8], uint32_t m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return m;
}

__device__ __forceinline__ void store8(int8_t* p, long long left, const float (&v)[8], const Divisor& s) {
  int q[8];
  if (s.usable()) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = (int)__builtin_rintf(s(v[j]));
  } else {
    // A scale of few units of 2^-149 may have been rounded down by up to a third: quotients past 127 are held there.
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = s.s > 0.0f ? (int)fminf(fmaxf(__builtin_rintf(v[j] / s.s), -127.0f), 127.0f) : 0;
  }
  if (left >= 8) {
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = (uint32_t)(q[4 * h] & 255) | (uint32_t)(q[4 * h + 1] & 255) << 8 | (uint32_t)(q[4 * h + 2] & 255) << 16 |
             (uint32_t)q[4 * h + 3] << 24;
    __builtin_memcpy(p, &w, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = (int8_t)q[j];
  }
}

// kWaves waves a row (with one, four rows a workgroup) by what a row's registers allow, kChunks groups of eight
// values a lane in registers; kChunks 0: any width, read a second time.
template <typename T, int kWaves, int kChunks>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void quantize_rows_kernel(
    const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scales, uint32_t rows, uint32_t width,
    uint32_t stride) {
  constexpr int kRows = kWaves == 1 ? 4 : 1, kLanes = 64 * kWaves;
  __shared__ uint32_t part[kWaves];
  const int lane = kWaves == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  for (unsigned long long row = (unsigned long long)blockIdx.x * kRows + (kWaves == 1 ? threadIdx.x >> 6 : 0);
       row < rows; row += (unsigned long long)gridDim.x * kRows) {
    const T* src = x + row * stride;
    int8_t* dst = q + row * width;
    float v[kChunks > 0 ? kChunks : 1][8];
    uint32_t m = 0;
    if constexpr (kChunks > 0) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const long long at = 8ll * (lane + kLanes * i);
        load8(src + min(at, (long long)width), (long long)width - at, v[i]);
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) m = max_bits(v[i], m);
    } else {
      for (long long at = 8ll * lane; at < width; at += 8ll * kLanes) {
        load8(src + at, (long long)width - at, v[0]);
        m = max_bits(v[0], m);
      }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if constexpr (kWaves > 1) {
      __syncthreads();  // the row before is done with the parts
      if ((lane & 63) == 0) part[lane >> 6] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = max(m, part[w]);
    }
    // A row with an infinity or a NaN: scale NaN, and zeros (s > 0 fails).
    const float s = m >= kInfBits ? __uint_as_float(0x7FC00000u) : __uint_as_float(m) / 127.0f;
    if (lane == 0) scales[row] = s;
    const Divisor d(s);
    if constexpr (kChunks > 0) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const long long at = 8ll * (lane + kLanes * i);
        if (at < width) store8(dst + at, (long long)width - at, v[i], d);
      }
    } else {
      for (long long at = 8ll * lane; at < width; at += 8ll * kLanes) {
        load8(src + at, (long long)width - at, v[0]);
        store8(dst + at, (long long)width - at, v[0], d);
      }
    }
  }
}

template <typename T>
hipError_t launch(const T* x, int8_t* q, float* scales, uint32_t rows, uint32_t width, uint32_t stride,
                  hipStream_t stream) {
  const unsigned one = (unsigned)std::min<uint64_t>(rows, 1u << 20), four = (unsigned)std::min<uint64_t>((rows + 3ull) / 4, 1u << 20);
#define ROWS(W, C, grid, block)                                                                              \
  hipLaunchKernelGGL((quantize_rows_kernel<T, W, C>), dim3(grid), dim3(block), 0, stream, x, q, scales, rows, \
                     width, stride)
  if (width <= 512)
    ROWS(1, 1, four, 256);
  else if (width <= 1024)
    ROWS(1, 2, four, 256);
  else if (width <= 2048)
    ROWS(4, 1, one, 256);
  else if (width <= 4096)
    ROWS(4, 2, one, 256);
  else if (width <= 8192)
    ROWS(4, 4, one, 256);
  else if (width <= 16384)
    ROWS(8, 4, one, 512);
  else
    ROWS(16, 0, one, 1024);
#undef ROWS
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_rows_int8(const void* x, bool bf16, int8_t* q, float* scales, uint32_t rows, uint32_t width,
                                     uint32_t stride, hipStream_t stream) {
  return bf16 ? launch(static_cast<const uint16_t*>(x), q, scales, rows, width, stride, stream)
              : launch(static_cast<const float*>(x), q, scales, rows, width, stride, stream);
}

}  // namespace prom
