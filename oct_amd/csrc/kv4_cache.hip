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
// lanes one token's head, both its keys and its values.  Bound by memory (25331
// rows of 8 heads of 128, bf16: write 26.4 us, 4.4 TB/s; read 24.5 us, 4.7 TB/s)
// and, for the few rows of a decode step, by the latency of the chain row ->
// sequence -> page -> store (64 rows: 5 us a launch).
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
// Exact: what the cache holds has eight significant bits, and is a multiple of 2^-132 (a step is one of 2^-131).
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

// The largest of eight neighbouring lanes.
__device__ __forceinline__ uint32_t max_of_8(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));   // the other of a pair
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));   // the other pair of four
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));  // mirrored within eight
}

// The IEEE quotient x / d for d of at most six significant bits, r = 1 / d to within a few ulps: q = fl(x r)
// is a few ulps off, the remainder q d - x has few enough bits to be exact, and x / d lies 2^-7 ulps or
// more from where rounding changes, far more than the error of q - remainder r.  The sign of a zero is kept.
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = x * r;
  return __builtin_fmaf(-__builtin_fmaf(q, d, -x), r, q);
}

// Step and codes of the eight channels v of a lane; the group's lanes are eight neighbours.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], uint32_t* param) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  m = max_of_8(m);
  const float top = __uint_as_float(m);
  // In this range nothing under- or overflows on the way to a quotient that is not rounded to zero.
  const bool plain = (top >= 0x1p-80f && top <= 0x1p80f) || m == 0;
  const bool all_plain = __all(plain);
  const uint32_t t = __float_as_uint(all_plain ? quotient(top, 6.0f, 1.0f / 6.0f) : top / 6.0f);
  const float s = __uint_as_float((t + 0x3FFFFu) & 0xFFFC0000u);
  const bool finite = m < kInfBits;
  *param = finite ? __float_as_uint(s) >> 16 : kNanParam;
  const bool some = finite && s > 0.0f;
  const float d = some ? s : 1.0f;
  float y[8];
  if (all_plain) {
    const float r = __builtin_amdgcn_rcpf(d);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = quotient(v[j], d, r);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = v[j] / d;
  }
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[0], y[1], 1.0f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], 1.0f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[4], y[5], 1.0f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[6], y[7], 1.0f, 3);
  return some ? codes : 0u;
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

// The sequences of rows, asked by a whole wave with one row at a time.  Up to 63 sequences: their starts
// are held by the lanes.  More: the answer before, where it still holds, or a search.
struct SequenceOf {
  const int32_t* starts;
  int n, held = 0, last = -1;
  bool few;
  __device__ __forceinline__ SequenceOf(const int32_t* starts_, int n_) : starts(starts_), n(n_), few(n_ < 64) {
    if (few) held = starts[min((int)threadIdx.x & 63, n)];
  }
  __device__ __forceinline__ int operator()(int r) {
    if (few) {
      const int at = __popcll(__ballot(((int)threadIdx.x & 63) <= n && held <= r)) - 1;
      return at < n ? at : -1;
    }
    if (last < 0 || r < starts[last] || r >= starts[last + 1]) last = find_sequence(starts, n, r);
    return last;
  }
};

// One item is a row's head, a wave holds 64 / (D / 8) items.  A workgroup takes one head of `take`
// neighbouring rows: what it writes of a page, whose codes and steps lie by head, are then whole lines
// but for the first and the last (heads of one row in neighbouring lanes: 36 us a write, 29 a read of
// 25331 rows of 8 heads of 128 in bf16).
template <typename T, int D, bool kWrite>
__global__ __launch_bounds__(256) void kv4_rows_kernel(const Kv4View c, T* k, T* v, const int32_t* __restrict__ starts,
                                                       uint32_t rows, uint32_t stride, uint32_t take) {
  constexpr int kLanes = D / 8, kItems = 64 / kLanes;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int j = lane % kLanes;
  SequenceOf sequence(starts, c.sequences);
  const unsigned long long blocks = (unsigned long long)((rows + take - 1) / take) * (uint32_t)c.kv_heads;
  for (unsigned long long block_id = blockIdx.x; block_id < blocks; block_id += gridDim.x) {
    const uint32_t part = (uint32_t)(block_id / (uint32_t)c.kv_heads);
    const uint32_t head = (uint32_t)(block_id - (unsigned long long)part * (uint32_t)c.kv_heads);
    const uint32_t to = min(rows, (part + 1) * take);
    for (uint32_t first = part * take + wave * kItems; first < to; first += 4 * kItems) {
      const uint32_t row = first + lane / kLanes;
      const size_t at = (size_t)row * stride + head * D + 8 * j;
      float x[8], y[8];
      if constexpr (kWrite) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
        if (row < to) {
          load8(k + at, x);
          load8(v + at, y);
        }
      }
      int seq = -1;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (first + i >= to) break;
        const int of = sequence((int)(first + i));
        if (lane / kLanes == i) seq = of;
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
      if constexpr (kWrite) {
        live = live && good;
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
}

template <typename T, bool kWrite>
hipError_t launch(const Kv4View& c, int head_dim, T* k, T* v, const int32_t* starts, uint32_t rows, uint32_t stride,
                  hipStream_t stream) {
  // Many rows: a page's length a workgroup; few: no more than its waves take at once (64 rows of 8 heads
  // of 128 would be 8 workgroups).
  const uint32_t least = 4 * (512 / (uint32_t)head_dim);
  const uint32_t take = (uint64_t)rows * c.kv_heads >= 2048 * 64 ? 64 : least;
  const uint64_t blocks = (uint64_t)((rows + take - 1) / take) * (uint32_t)c.kv_heads;
  const dim3 grid((unsigned)std::min<uint64_t>(blocks, 1u << 20));
#define ROWS(D)                                                                                             \
  case D:                                                                                                   \
    hipLaunchKernelGGL((kv4_rows_kernel<T, D, kWrite>), grid, dim3(256), 0, stream, c, k, v, starts, rows,  \
                       stride, take);                                                                       \
    break;
  switch (head_dim) {
    ROWS(64)
    ROWS(128)
    ROWS(256)
#undef ROWS
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
