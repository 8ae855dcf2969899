// The 4-bit weight matrix on the device, shared by what packs it (w4_matrix.hip) and what multiplies by it
// (gemm_w4.hip, moe_w4.hip).
//
// Tiles of 16 rows by 128 columns.  A tile's codes are 1 KiB, 16 bytes a lane of a wave: word s of lane l holds the
// codes of row l % 16, columns 32 s + 8 (l / 16) .. + 7, which is what that lane feeds into step s of four
// v_mfma_f32_16x16x32_bf16, so that one load brings a lane's operands of 128 columns and no lane needs another's.
// Tiles of a row of tiles follow each other: a wave that walks along K reads memory in order.  The steps lie behind
// all codes, tile by tile, [16][128 / group], so that a lane's steps of a tile are one load too.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace prom {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4TileN = 16, kW4TileK = 128, kW4TileBytes = kW4TileN * kW4TileK / 2;

// `count` matrices [n, k], `stride` bytes apart.
struct W4View {
  uint8_t* data;
  int n, k, group, count;
  int tiles_n, tiles_k;
  size_t stride;
};

inline W4View w4_view(void* data, uint32_t n, uint32_t k, uint32_t group, uint32_t count) {
  W4View w{static_cast<uint8_t*>(data), (int)n, (int)k, (int)group, (int)count, (int)((n + 15) / 16), (int)((k + 127) / 128), 0};
  w.stride = (size_t)w.tiles_n * w.tiles_k * (kW4TileBytes + 2 * kW4TileN * (kW4TileK / (size_t)group));
  return w;
}

#ifdef __HIPCC__
// Codes and steps of matrix e; kSteps = 128 / group.
__device__ __forceinline__ const u32x4* w4_codes(const W4View& w, int e, int tile_n) {
  return reinterpret_cast<const u32x4*>(w.data + e * w.stride + (size_t)tile_n * w.tiles_k * kW4TileBytes);
}
template <int kSteps>
__device__ __forceinline__ const uint16_t* w4_steps(const W4View& w, int e, int tile_n) {
  return reinterpret_cast<const uint16_t*>(w.data + e * w.stride + (size_t)w.tiles_n * w.tiles_k * kW4TileBytes) +
         (size_t)tile_n * w.tiles_k * (kW4TileN * kSteps);
}

// Eight codes as bf16 numbers (exact).
__device__ __forceinline__ bf16x8 w4_numbers(uint32_t codes) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
#endif

}  // namespace prom
