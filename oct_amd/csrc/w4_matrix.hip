// Weight matrices packed into 4 bits, and unpacked.
//
// A wave takes a tile of 16 rows by 128 columns (w4_tiles.h): it reads four rows at a time, eight columns a lane,
// so that a group's largest magnitude is a maximum over 4, 8 or 16 neighbouring lanes, and turns the words into the
// tile's order through LDS, so that codes leave as 16 bytes a lane; unpacking goes the other way.  Bound by memory: 16384x2048
// in bf16 packed in 19.4 us, 84 MB at 4.4 TB/s, unpacked in 13.5.
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

// Between a wave's LDS operations on words that only it uses: they are done in the program's order.
__device__ __forceinline__ void own_lds() { asm volatile("" ::: "memory"); }

template <typename T, int kGroup, bool kPack>
__global__ __launch_bounds__(256) void w4_tiles_kernel(const W4View w, T* __restrict__ rows, uint32_t stride) {
  constexpr int kSteps = kW4TileK / kGroup, kLanes = kGroup / 8;
  __shared__ uint32_t words[4][256];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int j = lane & 15;  // eight columns of a row
  const unsigned long long per = (unsigned long long)w.tiles_n * w.tiles_k, tiles = per * w.count;
  for (unsigned long long tile = 4ull * blockIdx.x + wave; tile < tiles; tile += 4ull * gridDim.x) {
    const int e = (int)(tile / per);
    const unsigned long long in = tile - e * per;
    const int tn = (int)(in / w.tiles_k), tk = (int)(in - (unsigned long long)tn * w.tiles_k);
    uint32_t* codes = reinterpret_cast<uint32_t*>(w.data + e * w.stride + in * kW4TileBytes);
    uint16_t* steps = reinterpret_cast<uint16_t*>(w.data + e * w.stride + per * kW4TileBytes) + in * (kW4TileN * kSteps);
    const int k = tk * kW4TileK + 8 * j, row = tn * kW4TileN + (lane >> 4);
    const bool whole = tn * kW4TileN + kW4TileN <= w.n && tk * kW4TileK + kW4TileK <= w.k;
    T* const at = rows + ((size_t)e * w.n + row) * stride + k;  // formed, not read, behind the last row or column
    float v[4][8];
    if constexpr (kPack) {
      // The four loads are on their way together where no row or column is missing.
      if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load8(at + (size_t)(4 * i) * stride, 8, v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) load8(at + (size_t)(4 * i) * stride, row + 4 * i < w.n ? w.k - k : 0, v[i]);
      }
      own_lds();  // the words of the tile before are read
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + (lane >> 4);
        uint32_t param;
        words[wave][tile_word(r, j)] = fp4_codes(v[i], max_of_lanes<kLanes>(max_bits(v[i])), &param);
        if (j % kLanes == 0) steps[r * kSteps + j / kLanes] = (uint16_t)param;
      }
      own_lds();
      reinterpret_cast<u32x4*>(codes)[lane] = *reinterpret_cast<const u32x4*>(&words[wave][4 * lane]);
    } else {
      const u32x4 mine = reinterpret_cast<const u32x4*>(codes)[lane];
      uint32_t step[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) step[i] = steps[(4 * i + (lane >> 4)) * kSteps + j / kLanes];
      own_lds();
      *reinterpret_cast<u32x4*>(&words[wave][4 * lane]) = mine;
      own_lds();
#pragma unroll
      for (int i = 0; i < 4; ++i) fp4_values(words[wave][tile_word(4 * i + (lane >> 4), j)], step[i], v[i]);
      if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store8(at + (size_t)(4 * i) * stride, 8, v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) store8(at + (size_t)(4 * i) * stride, row + 4 * i < w.n ? w.k - k : 0, v[i]);
      }
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
