// A mixture-of-experts layer of a few tokens on 4-bit weights:
//   l = x router^T, a token's experts the top_k largest l (ties to the lower expert), p their softmax weights,
//   out = sum_e p_e (act(x gate_e^T) * (x up_e^T)) down_e^T.
//
// Logits are sums in binary64 (a choice between two close experts does not depend on the order of a sum).  A pair
// is a token with one of its experts; an expert's pairs are the rows of its products (w4_product.h), read through a
// list, so that each reached expert's weights are read once for up to 64 pairs.  The hidden rows go between the two
// products as bf16 terms, in the form that the second one multiplies.
#include <algorithm>

#include "moe_w4.h"
#include "reactor_internal.h"
#include "w4_product.h"

namespace prom {
namespace {

// h as terms (see W4MoeArgs::hidden): bf16 rows carry 16 bits in two, fp32 rows 24 in three.
template <int kT>
struct W4RowsTerms {
  static constexpr int kTerms = kT;
  typedef uint16_t Element;
  struct Raw {
    u32x4 v[kT];
  };
  const uint16_t* p;
  size_t plane;
  bool live;
  template <bool kTail>
  __device__ __forceinline__ Raw fetch(int at, int k) const {
    Raw r{};
    if (!live) return r;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      if (!kTail || at + 8 <= k) {
        __builtin_memcpy(&r.v[t], p + t * plane + at, 16);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at + j < k) r.v[t][j >> 1] |= (uint32_t)p[t * plane + at + j] << (16 * (j & 1));
      }
    }
    return r;
  }
  __device__ __forceinline__ static void terms(const Raw& r, bf16x8 (&x)[kT]) {
#pragma unroll
    for (int t = 0; t < kT; ++t) x[t] = __builtin_bit_cast(bf16x8, r.v[t]);
  }
};

template <typename T>
struct Kind;
template <>
struct Kind<uint16_t> {
  typedef W4RowsBf16 Rows;
  static constexpr int kHiddenTerms = 2;
};
template <>
struct Kind<float> {
  typedef W4RowsF32 Rows;
  static constexpr int kHiddenTerms = 3;
};

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

__device__ __forceinline__ void put_terms(uint16_t* p, size_t plane, float v, uint16_t) {
  const __bf16 high = (__bf16)v;
  const float rest = __builtin_isfinite((float)high) ? v - (float)high : 0.0f;
  p[0] = __builtin_bit_cast(uint16_t, high);
  p[plane] = __builtin_bit_cast(uint16_t, (__bf16)rest);
}
__device__ __forceinline__ void put_terms(uint16_t* p, size_t plane, float v, float) {
  const uint32_t b = __float_as_uint(v);
  const float rest = __builtin_isinf(v) ? 0.0f : v - __uint_as_float(b & 0xFFFF0000u);
  const uint32_t c = __float_as_uint(rest);
  p[0] = (uint16_t)(b >> 16);
  p[plane] = (uint16_t)(c >> 16);
  p[2 * plane] = (uint16_t)(__float_as_uint(rest - __uint_as_float(c & 0xFFFF0000u)) >> 16);
}

// g sigmoid(g), or the tanh form of GELU, which is g sigmoid(2 sqrt(2/pi) (g + 0.044715 g^3)): the sigmoid keeps
// its relative precision where 1 + tanh cancels.
__device__ __forceinline__ float activation(float g, uint32_t kind) {
  const float z = kind == PROM_MOE_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g / (1.0f + expf(-z));
}

// ------------------------------------------------------------------ the router
template <typename T>
__global__ __launch_bounds__(256) void moe_logits_kernel(const W4MoeArgs a) {
  const int lane = (int)threadIdx.x & 63, e = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (e >= a.experts) return;
  const int hidden = a.gate.k;
  for (int t = (int)blockIdx.y; t < a.tokens; t += (int)gridDim.y) {
    const T* x = static_cast<const T*>(a.x) + (size_t)t * a.x_stride;
    const float* w = a.router + (size_t)e * hidden;
    double sum = 0.0;
    for (int c = lane; c < hidden; c += 64) sum += (double)value(x + c) * (double)w[c];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) a.logits[(size_t)t * a.experts + e] = sum;
  }
}

// Bit patterns in the order of the numbers; a NaN is below all of them.
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  if (v != v) return 1;
  return b >> 63 ? ~b : b | 1ull << 63;
}

// A wave a token: its experts, one after the other, and their weights.
__global__ __launch_bounds__(256) void moe_route_kernel(const W4MoeArgs a) {
  const int lane = (int)threadIdx.x & 63;
  const int t = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (t >= a.tokens) return;
  const double* l = a.logits + (size_t)t * a.experts;
  unsigned long long key[kMoeMaxExperts / 64];
  double top = 0.0, all = 0.0, chosen_sum = 0.0;
#pragma unroll
  for (int i = 0; i < kMoeMaxExperts / 64; ++i) key[i] = lane + 64 * i < a.experts ? order_of(l[lane + 64 * i]) : 0;
  double mine = 0.0;  // lane j: the j-th expert's weight before division
  int expert = 0;
  for (int j = 0; j < a.top_k; ++j) {
    unsigned long long best = 0;
    int at = 1 << 30;
#pragma unroll
    for (int i = 0; i < kMoeMaxExperts / 64; ++i)
      if (key[i] > best) best = key[i], at = lane + 64 * i;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const unsigned long long other = __shfl_xor(best, d);
      const int where = __shfl_xor(at, d);
      if (other > best || (other == best && where < at)) best = other, at = where;
    }
#pragma unroll
    for (int i = 0; i < kMoeMaxExperts / 64; ++i)
      if (lane + 64 * i == at) key[i] = 0;
    const double v = l[at];
    if (j == 0) top = v;
    const double p = exp(v - top);
    chosen_sum += p;
    if (lane == j) mine = p, expert = at;
  }
  if (!a.renormalise) {
    for (int e = lane; e < a.experts; e += 64) all += exp(l[e] - top);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d);
    chosen_sum = all;
  }
  if (lane < a.top_k) {
    const size_t pair = (size_t)t * a.top_k + lane;
    const float w = (float)(mine / chosen_sum);
    a.chosen[pair] = expert;
    a.weights[pair] = w;
    if (a.out_chosen != nullptr) a.out_chosen[pair] = expert;
    if (a.out_weights != nullptr) a.out_weights[pair] = w;
  }
}

// One workgroup: pairs by expert.  Where a pair lies in its expert's list does not change what is computed from it.
__global__ __launch_bounds__(1024) void moe_lists_kernel(const W4MoeArgs a) {
  __shared__ int count[kMoeMaxExperts], start[kMoeMaxExperts], slot[kMoeMaxExperts];
  static_assert(kMoeMaxExperts == 1024, "an expert a thread");
  const int e = (int)threadIdx.x, lane = e & 63, wave = e >> 6;
  const int pairs = a.tokens * a.top_k;
  count[e] = 0;
  __syncthreads();
  for (int p = e; p < pairs; p += 1024) atomicAdd(&count[a.chosen[p]], 1);
  __syncthreads();
  // Exclusive sums of pairs and of reached experts.
  const int c = count[e];
  int sum = c, some = c > 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int s = __shfl_up(sum, d), r = __shfl_up(some, d);
    if (lane >= d) sum += s, some += r;
  }
  __shared__ int wave_sum[16], wave_some[16];
  if (lane == 63) wave_sum[wave] = sum, wave_some[wave] = some;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += wave_sum[w], some += wave_some[w];
  start[e] = sum - c;
  if (c > 0) a.reached[some - 1] = MoeExpert{e, sum - c, c, 0};
  if (e == 1023) *a.reached_count = some;
  slot[e] = 0;
  __syncthreads();
  for (int p = e; p < pairs; p += 1024) {
    const int to = a.chosen[p];
    a.pairs[start[to] + atomicAdd(&slot[to], 1)] = p;
  }
}

// ------------------------------------------------------------------ the experts
// Hidden columns 16 blockIdx.x .. of one reached expert's pairs: gate and up sums, the activation, terms.
template <typename T, int kSteps, int kMT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void moe_hidden_kernel(const W4MoeArgs a) {
  typedef typename Kind<T>::Rows X;
  __shared__ float sums[kWaves][2 * kMT][4][64];
  if ((int)blockIdx.y >= *a.reached_count) return;
  const MoeExpert ex = a.reached[blockIdx.y];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = (int)blockIdx.x;
  const u32x4* const codes[2] = {w4_codes(a.gate, ex.expert, tile), w4_codes(a.up, ex.expert, tile)};
  const uint16_t* const steps[2] = {w4_steps<kSteps>(a.gate, ex.expert, tile), w4_steps<kSteps>(a.up, ex.expert, tile)};
  for (int first = 0; first < ex.count; first += 16 * kMT) {
    const int rows = min(ex.count - first, 16 * kMT);
    X x[kMT];
    floatx4 acc[kMT][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      const int r = 16 * m + (lane & 15);
      x[m].live = r < rows;
      const int pair = a.pairs[ex.start + first + min(r, rows - 1)];
      x[m].p = static_cast<const T*>(a.x) + (size_t)(pair / a.top_k) * a.x_stride;
      acc[m][0] = acc[m][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    w4_accumulate<kSteps, 2, kMT, 4>(codes, steps, x, (rows + 15) / 16, wave, a.gate.tiles_k, kWaves, a.gate.k, acc);
    if (first > 0) __syncthreads();  // the sums before are read
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][2 * m + i][r][lane] = acc[m][i][r];
    __syncthreads();
    for (int at = (int)threadIdx.x; at < kMT * 256; at += 64 * kWaves) {
      const int m = at >> 8, r = (at >> 6) & 3, l = at & 63;
      const int row = 16 * m + 4 * (l >> 4) + r, f = tile * kW4TileN + (l & 15);
      if (row >= rows || f >= a.gate.n) continue;
      float g = sums[0][2 * m][r][l], u = sums[0][2 * m + 1][r][l];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) g += sums[w][2 * m][r][l], u += sums[w][2 * m + 1][r][l];
      const int pair = a.pairs[ex.start + first + row];
      put_terms(a.hidden + (size_t)pair * a.hidden_stride + f, a.hidden_plane, activation(g, a.activation) * u, T());
    }
  }
}

// Output columns 16 blockIdx.x .. of one reached expert's pairs.
template <typename T, int kSteps, int kMT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void moe_down_kernel(const W4MoeArgs a) {
  typedef W4RowsTerms<Kind<T>::kHiddenTerms> X;
  __shared__ float sums[kWaves][kMT][4][64];
  if ((int)blockIdx.y >= *a.reached_count) return;
  const MoeExpert ex = a.reached[blockIdx.y];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = (int)blockIdx.x;
  const u32x4* const codes[1] = {w4_codes(a.down, ex.expert, tile)};
  const uint16_t* const steps[1] = {w4_steps<kSteps>(a.down, ex.expert, tile)};
  for (int first = 0; first < ex.count; first += 16 * kMT) {
    const int rows = min(ex.count - first, 16 * kMT);
    X x[kMT];
    floatx4 acc[kMT][1];
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      const int r = 16 * m + (lane & 15);
      x[m].live = r < rows;
      x[m].plane = a.hidden_plane;
      x[m].p = a.hidden + (size_t)a.pairs[ex.start + first + min(r, rows - 1)] * a.hidden_stride;
      acc[m][0] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    w4_accumulate<kSteps, 1, kMT, 4>(codes, steps, x, (rows + 15) / 16, wave, a.down.tiles_k, kWaves, a.down.k, acc);
    if (first > 0) __syncthreads();
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][m][r][lane] = acc[m][0][r];
    __syncthreads();
    for (int at = (int)threadIdx.x; at < kMT * 256; at += 64 * kWaves) {
      const int m = at >> 8, r = (at >> 6) & 3, l = at & 63;
      const int row = 16 * m + 4 * (l >> 4) + r, n = tile * kW4TileN + (l & 15);
      if (row >= rows || n >= a.down.n) continue;
      float v = sums[0][m][r][l];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += sums[w][m][r][l];
      a.part[(size_t)a.pairs[ex.start + first + row] * a.down.n + n] = v;
    }
  }
}

// out = sum over a token's experts, in their order, of weight times what they gave.
template <typename T>
__global__ __launch_bounds__(256) void moe_join_kernel(const W4MoeArgs a) {
  const unsigned long long count = (unsigned long long)a.tokens * (uint32_t)a.down.n;
  for (unsigned long long at = blockIdx.x * 256ull + threadIdx.x; at < count; at += gridDim.x * 256ull) {
    const unsigned long long t = at / (uint32_t)a.down.n;
    const uint32_t n = (uint32_t)(at - t * (uint32_t)a.down.n);
    float v = 0.0f;
    for (int j = 0; j < a.top_k; ++j) {
      const size_t pair = t * a.top_k + j;
      v = __builtin_fmaf(a.weights[pair], a.part[pair * (uint32_t)a.down.n + n], v);
    }
    put(static_cast<T*>(a.out) + t * a.out_stride + n, v);
  }
}

template <typename T, int kSteps, int kMT>
void launch_hidden(const W4MoeArgs& a, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kMT, 4>), grid, dim3(256), 0, stream, a);
}
template <typename T, int kSteps, int kMT>
void launch_down(const W4MoeArgs& a, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((moe_down_kernel<T, kSteps, kMT, 4>), grid, dim3(256), 0, stream, a);
}

template <typename T>
hipError_t launch(const W4MoeArgs& a, hipStream_t stream) {
  const int pairs = a.tokens * a.top_k, reached = std::min(a.experts, pairs);
  hipLaunchKernelGGL((moe_logits_kernel<T>), dim3((unsigned)(a.experts + 3) / 4, (unsigned)std::min(a.tokens, 4096)),
                     dim3(256), 0, stream, a);
  hipLaunchKernelGGL(moe_route_kernel, dim3((unsigned)(a.tokens + 3) / 4), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(moe_lists_kernel, dim3(1), dim3(1024), 0, stream, a);
  const dim3 hidden((unsigned)a.gate.tiles_n, (unsigned)reached), down((unsigned)a.down.tiles_n, (unsigned)reached);
#define STEPS(what, group, grid)                                                                     \
  switch (group) {                                                                                   \
    case 32:                                                                                         \
      a.tokens <= 16 ? launch_##what<T, 4, 1>(a, grid, stream) : launch_##what<T, 4, 4>(a, grid, stream); \
      break;                                                                                         \
    case 64:                                                                                         \
      a.tokens <= 16 ? launch_##what<T, 2, 1>(a, grid, stream) : launch_##what<T, 2, 4>(a, grid, stream); \
      break;                                                                                         \
    default:                                                                                         \
      a.tokens <= 16 ? launch_##what<T, 1, 1>(a, grid, stream) : launch_##what<T, 1, 4>(a, grid, stream); \
  }
  STEPS(hidden, a.gate.group, hidden)
  STEPS(down, a.down.group, down)
#undef STEPS
  const uint64_t count = (uint64_t)a.tokens * (uint32_t)a.down.n;
  hipLaunchKernelGGL((moe_join_kernel<T>), dim3((unsigned)std::min<uint64_t>((count + 255) / 256, 8192u)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace

size_t moe_w4_workspace(W4MoeArgs& a, bool bf16, void* base) {
  const size_t pairs = (size_t)a.tokens * a.top_k, experts = (size_t)a.experts;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* p = static_cast<char*>(base) + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  a.hidden_stride = (uint32_t)a.gate.tiles_n * kW4TileN;
  a.hidden_plane = pairs * a.hidden_stride;
  a.logits = reinterpret_cast<double*>(take((size_t)a.tokens * experts * sizeof(double)));
  a.chosen = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.weights = reinterpret_cast<float*>(take(pairs * sizeof(float)));
  a.pairs = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.reached = reinterpret_cast<MoeExpert*>(take(experts * sizeof(MoeExpert)));
  a.reached_count = reinterpret_cast<int32_t*>(take(sizeof(int32_t)));
  a.hidden = reinterpret_cast<uint16_t*>(take(a.hidden_plane * (bf16 ? 2 : 3) * sizeof(uint16_t)));
  a.part = reinterpret_cast<float*>(take(pairs * (size_t)a.down.n * sizeof(float)));
  return at;
}

hipError_t launch_moe_w4(const W4MoeArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<uint16_t>(a, stream) : launch<float>(a, stream);
}

}  // namespace prom
