// Weight matrices packed into 4 bits, and unpacked.
//
// A wave takes a tile of 16 rows by 128 columns (w4_tiles.h): it reads four rows at a time, eight columns a lane,
// so that a group's largest magnitude is a maximum over 4, 8 or 16 neighbouring lanes, and turns the words into the
// tile's order through LDS, so that codes leave as 16 bytes a lane.  Bound by memory.
#include "fp4_groups.h"
#include "reactor_internal.h"
#include "w4_tiles.h"

namespace prom {
namespace {

// Eight columns from p, any alignment of their type; zeros from the left-th on.
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
// Exact: a packed weight has eight significant bits.
__device__ __forceinline__ void store8(uint16_t* p, int left, const float (&v)[8]) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = (__float_as_uint(v[2 * j]) >> 16) | (__float_as_uint(v[2 * j + 1]) & 0xFFFF0000u);
  if (left >= 8) {
    __builtin_memcpy(p, &w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = (uint16_t)(j & 1 ? w[j >> 1] >> 16 : w[j >> 1]);
  }
}

// Where word j (columns 8 j .. 8 j + 7) of row r of a tile lies, in words.
__device__ __forceinline__ int tile_word(int r, int j) { return 4 * (16 * (j & 3) + r) + (j >> 2); }

template <typename T, int kGroup, bool kPack>
__global__ __launch_bounds__(256) void w4_tiles_kernel(const W4View w, T* __restrict__ rows, uint32_t stride) {
  constexpr int kSteps = kW4TileK / kGroup, kLanes = kGroup / 8;
  __shared__ uint32_t words[4][256];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int j = lane & 15;  // eight columns of a row
  const unsigned long long per = (unsigned long long)w.tiles_n * w.tiles_k, tiles = per * w.count;
  // Every wave of a workgroup makes the same number of rounds (barriers).
  for (unsigned long long first = 4ull * blockIdx.x; first < tiles; first += 4ull * gridDim.x) {
    const unsigned long long tile = first + wave;
    const bool live = tile < tiles;
    const int e = (int)((live ? tile : 0) / per);
    const unsigned long long in = (live ? tile : 0) - e * per;
    const int tn = (int)(in / w.tiles_k), tk = (int)(in - (unsigned long long)tn * w.tiles_k);
    uint32_t* codes = reinterpret_cast<uint32_t*>(w.data + e * w.stride + in * kW4TileBytes);
    uint16_t* steps = reinterpret_cast<uint16_t*>(w.data + e * w.stride + per * kW4TileBytes) + in * (kW4TileN * kSteps);
    const int k = tk * kW4TileK + 8 * j, left = w.k - k;
    if constexpr (!kPack) {
      u32x4 mine{};
      if (live) mine = reinterpret_cast<const u32x4*>(codes)[lane];
      *reinterpret_cast<u32x4*>(&words[wave][4 * lane]) = mine;
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + (lane >> 4), n = tn * kW4TileN + r;
      const bool inside = live && n < w.n && left > 0;
      T* at = rows + ((size_t)e * w.n + (inside ? n : 0)) * stride + (inside ? k : 0);
      float v[8];
      if constexpr (kPack) {
        load8(at, inside ? left : 0, v);
        uint32_t param;
        words[wave][tile_word(r, j)] = fp4_codes(v, max_of_lanes<kLanes>(max_bits(v)), &param);
        if (live && j % kLanes == 0) steps[r * kSteps + j / kLanes] = (uint16_t)param;
      } else if (inside) {
        fp4_values(words[wave][tile_word(r, j)], steps[r * kSteps + j / kLanes], v);
        store8(at, left, v);
      }
    }
    __syncthreads();
    if constexpr (kPack) {
      if (live) reinterpret_cast<u32x4*>(codes)[lane] = *reinterpret_cast<const u32x4*>(&words[wave][4 * lane]);
      __syncthreads();
    }
  }
}

template <typename T, bool kPack>
hipError_t launch(const W4View& w, T* rows, uint32_t stride, hipStream_t stream) {
  const uint64_t tiles = (uint64_t)w.tiles_n * w.tiles_k * w.count;
  const dim3 grid((unsigned)std::min<uint64_t>((tiles + 3) / 4, 1u << 20));
#define TILES(G)                                                                                                \
  case G:                                                                                                       \
    hipLaunchKernelGGL((w4_tiles_kernel<T, G, kPack>), grid, dim3(256), 0, stream, w, rows, stride);            \
    break;
  switch (w.group) {
    TILES(32)
    TILES(64)
    TILES(128)
#undef TILES
    default:
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_w4_pack(const W4View& w, const void* rows, bool bf16, uint32_t stride, hipStream_t stream) {
  void* r = const_cast<void*>(rows);
  return bf16 ? launch<uint16_t, true>(w, static_cast<uint16_t*>(r), stride, stream)
              : launch<float, true>(w, static_cast<float*>(r), stride, stream);
}

hipError_t launch_w4_unpack(const W4View& w, void* rows, bool bf16, uint32_t stride, hipStream_t stream) {
  return bf16 ? launch<uint16_t, false>(w, static_cast<uint16_t*>(rows), stride, stream)
              : launch<float, false>(w, static_cast<float*>(rows), stride, stream);
}

}  // namespace prom
