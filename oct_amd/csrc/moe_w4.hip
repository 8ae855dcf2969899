// A mixture-of-experts layer of a few tokens on 4-bit weights:
//   l = x router^T, a token's experts the top_k largest l (ties to the lower expert), p their softmax weights,
//   out = sum_e p_e (act(x gate_e^T) * (x up_e^T)) down_e^T.
//
// Three launches.  The router: a wave makes an expert's logits of four tokens, in binary64 (a choice between two close
// experts does not depend on the order of a sum); the last workgroup of four tokens' (tickets.h) chooses their experts, and
// the last of those lists the pairs, a token with one of its experts, by expert.  The hidden columns: a workgroup takes 16
// of one reached expert, its gate and up weights once for sixteen pairs at a time (w4_product.h), and leaves the hidden
// rows as bf16 terms, in the form that the second product multiplies.  The output columns: a workgroup takes 16 of all
// experts, its waves an expert (or a part of its K) each, weighs their sums and adds them by token in LDS.
#include <algorithm>

#include "moe_w4.h"
#include "reactor_internal.h"
#include "tickets.h"
#include "w4_product.h"

namespace prom {
namespace {

template <typename T>
struct Kind;
template <>
struct Kind<uint16_t> {
  typedef W4RowsBf16 Rows;
  static constexpr int kHiddenTerms = 2;  // 16 significant bits
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
constexpr int kTokenBlock = 4;
__device__ uint32_t moe_tickets[kMoeMaxPairs / kTokenBlock + 1];  // of blocks of tokens, and of the blocks
constexpr int kColumnTickets = 256;
__device__ uint32_t moe_column_tickets[kColumnTickets];

template <typename V>
__device__ __forceinline__ void store_agent(V* p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V load_agent(const V* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// v of another lane of the wave, 64 bits; 0 where there is none.
template <int kCtrl, int kRows>
__device__ __forceinline__ unsigned long long moved(unsigned long long v) {
  const int low = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRows, 0xF, false);
  const int high = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), kCtrl, kRows, 0xF, false);
  return (unsigned long long)(uint32_t)high << 32 | (uint32_t)low;
}
// The wave's v joined by `op`, whose neutral element is 0, in every lane: rows of sixteen by shifts of 1, 2, 4 and 8, then the
// rows by broadcasts of their last lanes.
template <typename F>
__device__ __forceinline__ unsigned long long wave_join(unsigned long long v, F&& op) {
  v = op(v, moved<0x111, 0xF>(v));
  v = op(v, moved<0x112, 0xF>(v));
  v = op(v, moved<0x114, 0xF>(v));
  v = op(v, moved<0x118, 0xF>(v));
  v = op(v, moved<0x142, 0xA>(v));
  v = op(v, moved<0x143, 0xC>(v));
  const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)v, 63);
  const uint32_t high = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63);
  return (unsigned long long)high << 32 | low;
}
__device__ __forceinline__ double wave_sum(double v) {
  return __longlong_as_double((long long)wave_join((unsigned long long)__double_as_longlong(v), [](auto a, auto b) {
    return (unsigned long long)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
  }));
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
  return wave_join(v, [](auto a, auto b) { return a > b ? a : b; });
}

// Bit patterns in the order of the numbers, 0 below all; a NaN is below every number.
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  if (v != v) return 1;
  return b >> 63 ? ~b : b | 1ull << 63;
}

// A wave chooses token t's experts, one after the other, and makes their weights; kMost logits a lane.
template <int kMost>
__device__ __forceinline__ void choose(const W4MoeArgs& a, int t) {
  const int lane = (int)threadIdx.x & 63;
  const double* l = a.logits + (size_t)t * a.experts;
  const int mine = (a.experts + 63) >> 6;
  double logit[kMost];
  unsigned long long key[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    key[i] = 0;
    logit[i] = 0.0;
    if (i < mine && lane + 64 * i < a.experts) {
      logit[i] = load_agent(l + lane + 64 * i);
      key[i] = order_of(logit[i]);
    }
  }
  double picked = 0.0, top = 0.0;  // lane j: the j-th expert's logit
  int expert = 0;
  for (int j = 0; j < a.top_k; ++j) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine) best = key[i] > best ? key[i] : best;
    best = wave_max(best);
    // The lowest expert that has it.
    bool found = false;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      if (i >= mine || found) continue;
      const unsigned long long has = __ballot(key[i] == best);
      if (has == 0) continue;
      found = true;
      const int at = __builtin_ctzll(has);
      const unsigned long long bits = (unsigned long long)__double_as_longlong(logit[i]);
      const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)bits, at);
      const uint32_t high = __builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), at);
      const double v = __longlong_as_double((long long)((unsigned long long)high << 32 | low));
      if (j == 0) top = v;
      if (lane == j) picked = v, expert = at + 64 * i;
      if (lane == at) key[i] = 0;
    }
  }
  const double p = lane < a.top_k ? exp(picked - top) : 0.0;
  double sum = p;
  if (!a.renormalise) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine && lane + 64 * i < a.experts) sum += exp(logit[i] - top);
  }
  sum = wave_sum(sum);
  if (lane < a.top_k) {
    const size_t pair = (size_t)t * a.top_k + lane;
    const float w = (float)(p / sum);
    store_agent(a.chosen + pair, expert);
    a.weights[pair] = w;
    if (a.out_chosen != nullptr) a.out_chosen[pair] = expert;
    if (a.out_weights != nullptr) a.out_weights[pair] = w;
  }
}

// A workgroup lists the pairs by expert.  Where a pair lies in its expert's list does not change what is computed from it.
__device__ __forceinline__ void list_pairs(const W4MoeArgs& a, int (&count)[kMoeMaxExperts], int (&start)[kMoeMaxExperts],
                                           int (&wave_sums)[2][4]) {
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int pairs = a.tokens * a.top_k, slots = min(a.experts, pairs);
  for (int e = tid; e < kMoeMaxExperts; e += 256) count[e] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += 256) atomicAdd(&count[load_agent(a.chosen + p)], 1);
  __syncthreads();
  // Four experts a thread: sums of pairs and of reached experts before them.
  int sum = 0, some = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = count[4 * tid + i];
    sum += c;
    some += c > 0;
  }
  const int own = sum, own_some = some;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int s = __shfl_up(sum, d), r = __shfl_up(some, d);
    if (lane >= d) sum += s, some += r;
  }
  if (lane == 63) wave_sums[0][wave] = sum, wave_sums[1][wave] = some;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) sum += wave_sums[0][w], some += wave_sums[1][w];
    all += wave_sums[1][w];
  }
  sum -= own;
  some -= own_some;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = count[4 * tid + i];
    start[4 * tid + i] = sum;
    if (c > 0) a.reached[some++] = MoeExpert{4 * tid + i, sum, c, 0};
    sum += c;
  }
  for (int s = all + tid; s < slots; s += 256) a.reached[s] = MoeExpert{0, 0, 0, 0};
  __syncthreads();
  for (int p = tid; p < pairs; p += 256) a.pairs[atomicAdd(&start[load_agent(a.chosen + p)], 1)] = p;
}

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) { __builtin_memcpy(v, p, 16); }
__device__ __forceinline__ void load4(const uint16_t* p, float (&v)[4]) {
  uint16_t w[4];
  __builtin_memcpy(w, p, 8);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float((uint32_t)w[j] << 16);
}

// grid.x: four experts each, a wave one; grid.y: blocks of tokens.
template <typename T, int kMost>
__global__ __launch_bounds__(256) void moe_router_kernel(const W4MoeArgs a) {
  __shared__ int count[kMoeMaxExperts], start[kMoeMaxExperts], wave_sums[2][4];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int e = (int)blockIdx.x * 4 + wave, hidden = a.gate.k;
  const int first = (int)blockIdx.y * kTokenBlock, tokens = min(a.tokens - first, kTokenBlock);
  if (e < a.experts) {
    const float* w = a.router + (size_t)e * hidden;
    const T* x[kTokenBlock];
    double sum[kTokenBlock];
#pragma unroll
    for (int t = 0; t < kTokenBlock; ++t) {
      x[t] = static_cast<const T*>(a.x) + (size_t)(first + min(t, tokens - 1)) * a.x_stride;
      sum[t] = 0.0;
    }
    const int whole = hidden & ~3;
#pragma unroll 4
    for (int c = 4 * lane; c < whole; c += 256) {
      float v[4];
      load4(w + c, v);
#pragma unroll
      for (int t = 0; t < kTokenBlock; ++t) {
        if (t > 0 && t >= tokens) break;
        float u[4];
        load4(x[t] + c, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[t] = __builtin_fma((double)u[j], (double)v[j], sum[t]);
      }
    }
    if (whole + lane < hidden)
#pragma unroll
      for (int t = 0; t < kTokenBlock; ++t)
        sum[t] = __builtin_fma((double)value(x[t] + whole + lane), (double)w[whole + lane], sum[t]);
#pragma unroll
    for (int t = 0; t < kTokenBlock; ++t) {
      if (t >= tokens) break;
      const double s = wave_sum(sum[t]);
      if (lane == 0) store_agent(a.logits + (size_t)(first + t) * a.experts + e, s);
    }
  }
  if (!last_to_arrive(&moe_tickets[1 + blockIdx.y], gridDim.x, &ticket)) return;
  if (wave < tokens) choose<kMost>(a, first + wave);
  if (!last_to_arrive(&moe_tickets[0], gridDim.y, &ticket)) return;
  list_pairs(a, count, start, wave_sums);
}

// ------------------------------------------------------------------ the experts
// Hidden columns 16 blockIdx.x .. of reached expert blockIdx.y: gate and up sums, the activation, terms.
template <typename T, int kSteps, W4Edge kEdge, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void moe_hidden_kernel(const W4MoeArgs a) {
  typedef typename Kind<T>::Rows X;
  __shared__ float sums[kWaves][2][4][64];
  const MoeExpert ex = a.reached[blockIdx.y];
  if (ex.count == 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = (int)blockIdx.x, tiles_k = a.gate.tiles_k;
  const u32x4* const codes[2] = {w4_codes(a.gate, ex.expert, tile), w4_codes(a.up, ex.expert, tile)};
  const uint16_t* const steps[2] = {w4_steps<kSteps>(a.gate, ex.expert, tile), w4_steps<kSteps>(a.up, ex.expert, tile)};
  for (int block = 0; block < ex.count; block += 16) {
    W4Tile<kSteps, 2> first;
    first.fetch(codes, steps, min(wave, tiles_k - 1));
    const int rows = min(ex.count - block, 16);
    const int mine = a.pairs[ex.start + block + min(lane & 15, rows - 1)];
    X x[1];
    x[0].p = static_cast<const T*>(a.x) + (size_t)((unsigned)mine / (unsigned)a.top_k) * a.x_stride;
    floatx4 acc[1][2] = {};
    w4_accumulate<kSteps, 2, 1, kEdge>(codes, steps, first, x, wave, tiles_k, kWaves, a.gate.k, acc);
    if (block > 0) __syncthreads();  // the sums before are read
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][i][r][lane] = acc[0][i][r];
    __syncthreads();
    for (int at = (int)threadIdx.x; at < rows * 16; at += 64 * kWaves) {
      const int row = at >> 4, f = tile * kW4TileN + (at & 15), r = row & 3, l = 16 * (row >> 2) + (at & 15);
      float g = sums[0][0][r][l], u = sums[0][1][r][l];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) g += sums[w][0][r][l], u += sums[w][1][r][l];
      const int pair = a.pairs[ex.start + block + row];
      // Columns behind the last are zeros: whole tiles are multiplied.
      const float h = f < a.gate.n ? activation(g, a.activation) * u : 0.0f;
      uint16_t* to = a.hidden + (size_t)pair * a.hidden_stride + f;
      put_terms(to, a.hidden_plane, h, T());
      if (tile == a.gate.tiles_n - 1)
        for (uint32_t c = (uint32_t)f + 16; c < a.hidden_stride; c += 16)
          put_terms(a.hidden + (size_t)pair * a.hidden_stride + c, a.hidden_plane, 0.0f, T());
    }
  }
}

constexpr int kFewTokens = 64;

// Output columns 16 blockIdx.x .. of up to kFewTokens tokens.  A unit is a part of K of a reached expert; slice y of them
// is dealt to the waves.
template <typename T, int kSteps, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void moe_out_kernel(const W4MoeArgs a) {
  typedef W4RowsTerms<Kind<T>::kHiddenTerms> X;
  __shared__ float sums[kWaves][kFewTokens][16];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = (int)blockIdx.x, tiles_k = a.down.tiles_k, slots = min(a.experts, a.tokens * a.top_k);
  const int count = a.tokens * 16;
  for (int at = lane; at < count; at += 64) sums[wave][at >> 4][at & 15] = 0.0f;  // each wave its own
  for (int unit = (int)blockIdx.y * kWaves + wave; unit < slots * a.split; unit += kWaves * a.slices) {
    const int slot = unit / a.split, part = unit - slot * a.split;
    const MoeExpert ex = a.reached[slot];
    if (ex.count == 0) break;  // nor are there any behind it
    const u32x4* const codes[1] = {w4_codes(a.down, ex.expert, tile)};
    const uint16_t* const steps[1] = {w4_steps<kSteps>(a.down, ex.expert, tile)};
    const int begin = tiles_k * part / a.split, end = tiles_k * (part + 1) / a.split;
    if (begin == end) continue;
    for (int block = 0; block < ex.count; block += 16) {
      W4Tile<kSteps, 1> first;
      first.fetch(codes, steps, begin);
      const int rows = min(ex.count - block, 16);
      const int mine = a.pairs[ex.start + block + min(lane & 15, rows - 1)];
      const float weight = a.weights[mine];
      X x[1];
      x[0].plane = a.hidden_plane;
      x[0].p = a.hidden + (size_t)mine * a.hidden_stride;
      floatx4 acc[1][1] = {};
      w4_accumulate<kSteps, 1, 1, kEdgeNone>(codes, steps, first, x, begin, end, 1, a.down.k, acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // Row 4 (lane / 16) + r: its pair and weight are with the lane of that number.
        const int row = 4 * (lane >> 4) + r;
        const int token = (int)((unsigned)__shfl(mine, row) / (unsigned)a.top_k);
        const float p = __shfl(weight, row);
        if (row < rows) sums[wave][token][lane & 15] += p * acc[0][0][r];
      }
    }
  }
  __syncthreads();
  const int column0 = tile * kW4TileN;
  T* out = static_cast<T*>(a.out) + column0;
  float* part = a.part + ((size_t)tile * a.slices) * (kFewTokens * 16);
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    float v = sums[0][at >> 4][at & 15];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][at >> 4][at & 15];
    if (a.slices > 1)
      store_agent(part + (size_t)blockIdx.y * (kFewTokens * 16) + at, v);
    else if (column0 + (at & 15) < a.down.n)
      put(out + (size_t)(at >> 4) * a.out_stride + (at & 15), v);
  }
  if (a.slices == 1 || !last_to_arrive(&moe_column_tickets[tile], (uint32_t)a.slices, &ticket)) return;
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    float v = load_agent(part + at);
    for (int s = 1; s < a.slices; ++s) v += load_agent(part + (size_t)s * (kFewTokens * 16) + at);
    if (column0 + (at & 15) < a.down.n) put(out + (size_t)(at >> 4) * a.out_stride + (at & 15), v);
  }
}

// More tokens: output columns 16 blockIdx.x .. of reached expert blockIdx.y's pairs, and their sums by token.
template <typename T, int kSteps>
__global__ __launch_bounds__(256) void moe_down_kernel(const W4MoeArgs a) {
  typedef W4RowsTerms<Kind<T>::kHiddenTerms> X;
  __shared__ float sums[4][4][64];
  const MoeExpert ex = a.reached[blockIdx.y];
  if (ex.count == 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = (int)blockIdx.x, tiles_k = a.down.tiles_k;
  const u32x4* const codes[1] = {w4_codes(a.down, ex.expert, tile)};
  const uint16_t* const steps[1] = {w4_steps<kSteps>(a.down, ex.expert, tile)};
  for (int block = 0; block < ex.count; block += 16) {
    W4Tile<kSteps, 1> first;
    first.fetch(codes, steps, min(wave, tiles_k - 1));
    const int rows = min(ex.count - block, 16);
    X x[1];
    x[0].plane = a.hidden_plane;
    x[0].p = a.hidden + (size_t)a.pairs[ex.start + block + min(lane & 15, rows - 1)] * a.hidden_stride;
    floatx4 acc[1][1] = {};
    w4_accumulate<kSteps, 1, 1, kEdgeNone>(codes, steps, first, x, wave, tiles_k, 4, a.down.k, acc);
    if (block > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][r][lane] = acc[0][0][r];
    __syncthreads();
    const int row = (int)threadIdx.x >> 4, n = tile * kW4TileN + ((int)threadIdx.x & 15);
    const int r = row & 3, l = 16 * (row >> 2) + ((int)threadIdx.x & 15);
    if (row < rows && n < a.down.n)
      a.part[(size_t)a.pairs[ex.start + block + row] * a.down.n + n] =
          sums[0][r][l] + sums[1][r][l] + sums[2][r][l] + sums[3][r][l];
  }
}

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

template <typename T, int kSteps>
void launch_hidden(const W4MoeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.gate.tiles_n, (unsigned)std::min(a.experts, a.tokens * a.top_k));
  if (a.gate.k % kW4TileK == 0)
    hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kEdgeNone, 4>), grid, dim3(256), 0, stream, a);
  else if (a.gate.k >= 8)
    hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kEdgeShift, 4>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kEdgeShort, 4>), grid, dim3(256), 0, stream, a);
}

template <typename T, int kSteps>
void launch_out(const W4MoeArgs& a, hipStream_t stream) {
  if (a.tokens <= kFewTokens) {
    hipLaunchKernelGGL((moe_out_kernel<T, kSteps, 8>), dim3((unsigned)a.down.tiles_n, (unsigned)a.slices), dim3(512), 0,
                       stream, a);
    return;
  }
  hipLaunchKernelGGL((moe_down_kernel<T, kSteps>),
                     dim3((unsigned)a.down.tiles_n, (unsigned)std::min(a.experts, a.tokens * a.top_k)), dim3(256), 0, stream, a);
  const uint64_t count = (uint64_t)a.tokens * (uint32_t)a.down.n;
  hipLaunchKernelGGL((moe_join_kernel<T>), dim3((unsigned)std::min<uint64_t>((count + 255) / 256, 8192u)), dim3(256), 0,
                     stream, a);
}

template <typename T>
hipError_t launch(const W4MoeArgs& a, hipStream_t stream) {
  const dim3 router((unsigned)(a.experts + 3) / 4, (unsigned)(a.tokens + kTokenBlock - 1) / kTokenBlock);
  if (a.experts <= 64)
    hipLaunchKernelGGL((moe_router_kernel<T, 1>), router, dim3(256), 0, stream, a);
  else if (a.experts <= 256)
    hipLaunchKernelGGL((moe_router_kernel<T, 4>), router, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((moe_router_kernel<T, 16>), router, dim3(256), 0, stream, a);
#define STEPS(what, group) \
  if (group == 32)         \
    what<T, 4>(a, stream); \
  else if (group == 64)    \
    what<T, 2>(a, stream); \
  else                     \
    what<T, 1>(a, stream);
  STEPS(launch_hidden, a.gate.group)
  STEPS(launch_out, a.down.group)
#undef STEPS
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
  const int slots = (int)std::min(experts, pairs);
  a.split = 1;
  a.slices = 1;
  while (a.split < 4 && slots * a.split < 16 && a.down.tiles_k >= 4 * a.split) a.split *= 2;
  while (a.slices < 8 && a.down.tiles_n * a.slices < 256 && slots * a.split >= 16 * a.slices) a.slices *= 2;
  a.hidden_stride = (uint32_t)a.down.tiles_k * kW4TileK;
  a.hidden_plane = pairs * a.hidden_stride;
  a.logits = reinterpret_cast<double*>(take((size_t)a.tokens * experts * sizeof(double)));
  a.chosen = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.weights = reinterpret_cast<float*>(take(pairs * sizeof(float)));
  a.pairs = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.reached = reinterpret_cast<MoeExpert*>(take((size_t)slots * sizeof(MoeExpert)));
  a.hidden = reinterpret_cast<uint16_t*>(take(a.hidden_plane * (bf16 ? 2 : 3) * sizeof(uint16_t)));
  const size_t parts = a.tokens <= kFewTokens ? (size_t)a.down.tiles_n * a.slices * (kFewTokens * 16) : pairs * (size_t)a.down.n;
  a.part = reinterpret_cast<float*>(take(parts * sizeof(float)));
  return at;
}

hipError_t launch_moe_w4(const W4MoeArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<uint16_t>(a, stream) : launch<float>(a, stream);
}

}  // namespace prom
