// The product with 4-bit weights: c[i, j] = sum_k x[i, k] w[j, k], w as w4_tiles.h lays it out.
//
// Few rows: bound by reading w.  A workgroup takes kNT tiles of 16 columns, its waves every kWaves-th tile of K
// each (memory is read in order by the workgroup), and adds their sums through LDS; where columns are few, K is cut into
// slices over workgroups too, whose sums a second kernel adds in order.
#include <algorithm>

#include "reactor_internal.h"
#include "w4_product.h"

namespace prom {
namespace {

struct W4Args {
  W4View w;
  const void* x;
  void* out;
  float* part;  // slices' sums [slices][m][n] (null: one slice)
  uint32_t x_stride, out_stride;
  int m, slices;
};

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

template <typename X, int kSteps, int kNT, int kMT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void w4_rows_kernel(const W4Args a) {
  typedef typename X::Element T;
  __shared__ float sums[kWaves][kMT * kNT][4][64];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row0 = (int)blockIdx.z * (16 * kMT), rows = min(a.m - row0, 16 * kMT);
  X x[kMT];
#pragma unroll
  for (int m = 0; m < kMT; ++m) {
    const int r = 16 * m + (lane & 15);
    x[m].live = r < rows;
    x[m].p = static_cast<const T*>(a.x) + (size_t)(row0 + min(r, rows - 1)) * a.x_stride;
  }
  const u32x4* codes[kNT];
  const uint16_t* steps[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    const int tile = min((int)blockIdx.x * kNT + i, a.w.tiles_n - 1);
    codes[i] = w4_codes(a.w, 0, tile);
    steps[i] = w4_steps<kSteps>(a.w, 0, tile);
  }
  floatx4 acc[kMT][kNT];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int i = 0; i < kNT; ++i) acc[m][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  // Slice y of K: tiles begin .. end - 1.
  const int slice = (int)blockIdx.y;
  const int begin = (int)((long long)a.w.tiles_k * slice / a.slices);
  const int end = (int)((long long)a.w.tiles_k * (slice + 1) / a.slices);
  w4_accumulate<kSteps, kNT, kMT, 4>(codes, steps, x, (rows + 15) / 16, begin + wave, end, kWaves, a.w.k, acc);
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][m * kNT + i][r][lane] = acc[m][i][r];
  __syncthreads();
  for (int at = (int)threadIdx.x; at < kMT * kNT * 256; at += 64 * kWaves) {
    const int tile = at >> 8, r = (at >> 6) & 3, l = at & 63;
    const int row = 16 * (tile / kNT) + 4 * (l >> 4) + r;
    const int column = ((int)blockIdx.x * kNT + tile % kNT) * kW4TileN + (l & 15);
    if (row >= rows || column >= a.w.n) continue;
    float v = sums[0][tile][r][l];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][tile][r][l];
    if (a.part != nullptr)
      a.part[((size_t)slice * a.m + row0 + row) * a.w.n + column] = v;
    else
      put(static_cast<T*>(a.out) + (size_t)(row0 + row) * a.out_stride + column, v);
  }
}

// out = the sum of the slices in order.
template <typename T>
__global__ __launch_bounds__(256) void w4_slices_kernel(const W4Args a) {
  const unsigned long long count = (unsigned long long)a.m * a.w.n;
  for (unsigned long long at = blockIdx.x * 256ull + threadIdx.x; at < count; at += gridDim.x * 256ull) {
    float v = a.part[at];
    for (int s = 1; s < a.slices; ++s) v += a.part[s * count + at];
    const unsigned long long row = at / (uint32_t)a.w.n;
    put(static_cast<T*>(a.out) + row * a.out_stride + (at - row * (uint32_t)a.w.n), v);
  }
}

struct W4Plan {
  int nt, mt, waves, slices;
};

W4Plan plan_w4(uint32_t m, const W4View& w) {
  W4Plan p{1, m <= 16 ? 1 : m <= 32 ? 2 : 4, 4, 1};
  if (w.tiles_k > 32) p.waves = 8;
  while (p.slices < 8 && w.tiles_n * p.slices < 256 && w.tiles_k >= 16 * p.slices * p.waves) p.slices *= 2;
  return p;
}

template <typename X, int kSteps>
hipError_t launch_steps(const W4Plan& p, const W4Args& a, hipStream_t stream) {
  typedef typename X::Element T;
  const dim3 grid((unsigned)((a.w.tiles_n + p.nt - 1) / p.nt), (unsigned)a.slices,
                  (unsigned)((a.m + 16 * p.mt - 1) / (16 * p.mt)));
#define ROWS(NT, MT, W)                                                                                             \
  if (p.nt == NT && p.mt == MT && p.waves == W)                                                                     \
    hipLaunchKernelGGL((w4_rows_kernel<X, kSteps, NT, MT, W>), grid, dim3(64 * W), 0, stream, a);
  ROWS(1, 1, 4) ROWS(1, 1, 8) ROWS(1, 2, 4) ROWS(1, 2, 8) ROWS(1, 4, 4) ROWS(1, 4, 8)
#undef ROWS
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.part == nullptr) return e;
  const uint64_t count = (uint64_t)a.m * (uint32_t)a.w.n;
  hipLaunchKernelGGL((w4_slices_kernel<T>), dim3((unsigned)std::min<uint64_t>((count + 255) / 256, 8192u)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

template <typename X>
hipError_t launch(const W4Plan& p, const W4Args& a, hipStream_t stream) {
  switch (a.w.group) {
    case 32:
      return launch_steps<X, 4>(p, a, stream);
    case 64:
      return launch_steps<X, 2>(p, a, stream);
    case 128:
      return launch_steps<X, 1>(p, a, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_gemm_w4(const W4View& w, const void* x, uint32_t x_stride, void* out, uint32_t out_stride, bool bf16,
                          uint32_t m, hipStream_t stream) {
  W4Args a{w, x, out, nullptr, x_stride, out_stride, (int)m, 1};
  const W4Plan p = plan_w4(m, w);
  if (p.slices > 1) {
    a.part = static_cast<float*>(staging(6, (size_t)p.slices * m * (uint32_t)w.n * sizeof(float)));
    if (a.part != nullptr) a.slices = p.slices;
  }
  return bf16 ? launch<W4RowsBf16>(p, a, stream) : launch<W4RowsF32>(p, a, stream);
}

}  // namespace prom
