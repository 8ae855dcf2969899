// Keys and values quantised to 4 bits as they are written to a paged cache, and
// read back.
//
// A group of 64 channels of one token's head has a step s = max |x| / 6, rounded
// up to six significant bits, and per channel an E2M1 number (0, 1/2, 1, 3/2, 2,
// 3, 4, 6 and negatives): s times that has eight significant bits, so that fp32
// and bf16 hold what is read back exactly, and the hardware turns two codes into
// two bf16 or fp32 numbers in one instruction.  x / s is the IEEE quotient and
// the conversion rounds halves to the even code: the codes are the definition's,
// bit for bit.
//
// A lane handles eight channels (one 4-byte word of codes), a group of D / 8
// lanes one token's head, both its keys and its values.  Bound by memory and, for
// the few rows of a decode step, by the latency of the chain row -> sequence ->
// page -> store.
#include "reactor_internal.h"

namespace prom {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kInfBits = 0x7F800000u;
constexpr uint32_t kNanParam = 0x7FC0u;

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) { __builtin_memcpy(v, p, 32); }
__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
  u32x4 w;
  __builtin_memcpy(&w, p, 16);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) { __builtin_memcpy(p, v, 32); }
// Exact: what the cache holds has eight significant bits (a step near fp32's smallest
// numbers, whose low bits bf16 drops, aside: these are rounded toward zero).
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = (__float_as_uint(v[2 * j]) >> 16) | (__float_as_uint(v[2 * j + 1]) & 0xFFFF0000u);
  __builtin_memcpy(p, &w, 16);
}

// Where word j (channels 8 j .. 8 j + 7) of a key row lies.
template <int D>
__device__ __forceinline__ int key_word(int j) {
  if constexpr (D == 64) return 2 * (j & 3) + (j >> 2);
  return (j & ~15) + 4 * (j & 3) + ((j >> 2) & 3);
}

// Step and codes of the eight channels v of a lane; the group's lanes are eight neighbours.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], uint32_t* param) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  const uint32_t t = __float_as_uint(__uint_as_float(m) / 6.0f);
  const float s = __uint_as_float((t + 0x3FFFFu) & 0xFFFC0000u);
  const bool finite = m < kInfBits;
  *param = finite ? __float_as_uint(s) >> 16 : kNanParam;
  const bool some = finite && s > 0.0f;
  uint32_t codes = 0;
  float y[8];
  const Divisor by(some ? s : 1.0f);
  if (__all(by.usable())) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = some ? __builtin_copysignf(by(v[j]), v[j]) : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = some ? v[j] / s : 0.0f;
  }
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[0], y[1], 1.0f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], 1.0f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[4], y[5], 1.0f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[6], y[7], 1.0f, 3);
  return codes;
}

__device__ __forceinline__ void values8(uint32_t codes, uint32_t param, float (&v)[8]) {
  const float s = __uint_as_float(param << 16);
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const floatx2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const floatx2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  v[0] = a.x * s, v[1] = a.y * s, v[2] = b.x * s, v[3] = b.y * s;
  v[4] = c.x * s, v[5] = c.y * s, v[6] = d.x * s, v[7] = d.y * s;
}

// One item is a row's head.  A wave holds 64 / (D / 8) neighbouring items, heads
// fastest, so that loads of neighbouring lanes are neighbours in memory.
template <typename T, int D, bool kWrite>
__global__ __launch_bounds__(256) void kv4_rows_kernel(const Kv4View c, T* k, T* v, const int32_t* __restrict__ starts,
                                                       uint32_t rows, uint32_t stride) {
  constexpr int kLanes = D / 8, kItems = 64 / kLanes;
  const int lane = (int)threadIdx.x & 63;
  const int j = lane % kLanes;
  const unsigned long long items = (unsigned long long)rows * (uint32_t)c.kv_heads;
  const unsigned long long waves = (unsigned long long)gridDim.x * 4;
  for (unsigned long long first = ((unsigned long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * kItems; first < items;
       first += waves * kItems) {
    // The sequences of the wave's items, one search after another with all 64 lanes.
    uint32_t row = 0, head = 0;
    int seq = -1, last = -1, last_seq = -1;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const unsigned long long item = first + i;
      if (item >= items) break;
      const uint32_t r = (uint32_t)(item / (uint32_t)c.kv_heads);
      if ((int)r != last) {
        last_seq = find_sequence(starts, c.sequences, (int)r);
        last = (int)r;
      }
      if (lane / kLanes == i) {
        row = r;
        head = (uint32_t)(item - (unsigned long long)r * (uint32_t)c.kv_heads);
        seq = last_seq;
      }
    }
    // Lanes of a group agree; a group without a place passes through the shuffles idly.
    long long token = -1;
    if (seq >= 0) token = (long long)c.lengths[seq] - (starts[seq + 1] - (long long)row);
    bool live = token >= 0;
    const long long place = token >> 6;
    uint32_t page = 0xFFFFFFFFu;
    if (live && place < c.table_stride) page = (uint32_t)c.table[(size_t)seq * c.table_stride + place];
    const bool good = page < c.pages;
    const int slot = (int)(token & 63);
    uint8_t* block = c.pool + ((size_t)(good ? page : 0u) * c.kv_heads + head) * kv4_block_bytes(D);
    uint32_t* key = reinterpret_cast<uint32_t*>(block + slot * (D / 2)) + key_word<D>(j);
    uint32_t* value = reinterpret_cast<uint32_t*>(block + kKv4Page * D / 2 + slot * (D / 2)) + j;
    uint16_t* params = reinterpret_cast<uint16_t*>(block + kKv4Page * D) + (j >> 3) * kKv4Page + slot;
    constexpr int kValueParams = D / 64 * kKv4Page;
    const size_t at = (size_t)row * stride + head * D + 8 * j;
    float x[8];
    if constexpr (kWrite) {
      live = live && good;
      float y[8] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
      if (live) {
        load8(k + at, x);
        load8(v + at, y);
      }
      uint32_t kp, vp;
      const uint32_t kc = quantise8(x, &kp), vc = quantise8(y, &vp);
      if (live) {
        *key = kc;
        *value = vc;
        if ((j & 7) == 0) {
          params[0] = (uint16_t)kp;
          params[kValueParams] = (uint16_t)vp;
        }
      }
    } else if (live) {
      if (k != nullptr) {
        values8(good ? *key : 0u, good ? params[0] : kNanParam, x);
        store8(k + at, x);
      }
      if (v != nullptr) {
        values8(good ? *value : 0u, good ? params[kValueParams] : kNanParam, x);
        store8(v + at, x);
      }
    }
  }
}

template <typename T, bool kWrite>
hipError_t launch(const Kv4View& c, int head_dim, T* k, T* v, const int32_t* starts, uint32_t rows, uint32_t stride,
                  hipStream_t stream) {
  const uint64_t items = (uint64_t)rows * c.kv_heads, a_block = 4 * (512 / head_dim);
  const unsigned grid = (unsigned)std::min<uint64_t>((items + a_block - 1) / a_block, 1u << 20);
  switch (head_dim) {
    case 64:
      hipLaunchKernelGGL((kv4_rows_kernel<T, 64, kWrite>), dim3(grid), dim3(256), 0, stream, c, k, v, starts, rows, stride);
      break;
    case 128:
      hipLaunchKernelGGL((kv4_rows_kernel<T, 128, kWrite>), dim3(grid), dim3(256), 0, stream, c, k, v, starts, rows, stride);
      break;
    case 256:
      hipLaunchKernelGGL((kv4_rows_kernel<T, 256, kWrite>), dim3(grid), dim3(256), 0, stream, c, k, v, starts, rows, stride);
      break;
    default:
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_write(const Kv4View& c, int head_dim, const void* k, const void* v, bool bf16,
                            const int32_t* row_starts, uint32_t rows, uint32_t stride, hipStream_t stream) {
  void* kk = const_cast<void*>(k);
  void* vv = const_cast<void*>(v);
  return bf16 ? launch<uint16_t, true>(c, head_dim, static_cast<uint16_t*>(kk), static_cast<uint16_t*>(vv), row_starts,
                                       rows, stride, stream)
              : launch<float, true>(c, head_dim, static_cast<float*>(kk), static_cast<float*>(vv), row_starts, rows,
                                    stride, stream);
}

hipError_t launch_kv4_read(const Kv4View& c, int head_dim, void* k, void* v, bool bf16, const int32_t* row_starts,
                           uint32_t rows, uint32_t stride, hipStream_t stream) {
  return bf16 ? launch<uint16_t, false>(c, head_dim, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), row_starts,
                                        rows, stride, stream)
              : launch<float, false>(c, head_dim, static_cast<float*>(k), static_cast<float*>(v), row_starts, rows,
                                     stride, stream);
}

}  // namespace prom
