// A mixture-of-experts layer of a few tokens on 4-bit weights:
//   l = x router^T, a token's experts the top_k largest l (ties to the lower expert), p their softmax weights,
//   out = sum_e p_e (act(x gate_e^T) * (x up_e^T)) down_e^T.
//
// Three launches.  The router: a wave makes an expert's logits of two tokens, in binary64 (a choice between two close
// experts does not depend on the order of a sum); the last workgroup of two tokens' (tickets.h) chooses their experts.  The
// hidden columns: a workgroup takes 32 of one reached expert, its gate and up weights once for sixteen pairs, a token with
// one of its experts (w4_product.h), and leaves the hidden rows as bf16 terms, in the form that the second product
// multiplies.  The output columns: a wave takes 32 or 64 of an expert (or of a part of its K) and leaves its sums by pair;
// the last workgroup of those columns weighs and joins them in the order of a token's experts.  Up to 64 tokens each wave
// looks up itself which of them chose its expert; above, the router's last workgroup lists the pairs by expert, and the
// sums are joined in a fourth launch.
//
// Bound by the reached experts' weights, and for a token by the latency of three kernels that follow one another.  64
// experts of 1024 with 2048 outer columns, 8 a token, in bf16: a token 4.7 + 6.1 + 7.6 us (28 MB at 2.0 TB/s in the last
// two), 64 tokens, which reach all experts, 9.9 + 33.2 + 29.7 us (214 MB at 3.4 TB/s; 64 rows of x and of the hidden
// columns come from L2 for each workgroup).
#include <algorithm>

#include "moe_w4.h"
#include "reactor_internal.h"
#include "tickets.h"
#include "w4_product.h"
#include "wave_ops.h"

namespace prom {
namespace {

template <typename T>
struct Kind;
template <>
struct Kind<uint16_t> {
  typedef W4RowsBf16 Rows;
};
template <>
struct Kind<float> {
  typedef W4RowsF32 Rows;
};
// A hidden value's bf16 terms: all of fp32's bits (two terms, sixteen bits, moved a bf16 result by 1.1e-4 to 2.3e-4 of its
// size, as its roundings fell another way).
constexpr int kHiddenTerms = 3;

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

// The upper half of what the ones before leave, as w4_split; an infinity is its first term.
__device__ __forceinline__ void put_terms(uint16_t* p, size_t plane, float v) {
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
constexpr int kTokenBlock = 2;
__device__ uint32_t moe_tickets[kMoeMaxPairs / kTokenBlock + 1];  // of blocks of tokens, and of the blocks
constexpr int kColumnTickets = 1024;
constexpr int kHiddenTiles = 2, kHiddenWaves = 4, kOutWaves = 8;
__device__ uint32_t moe_column_tickets[kColumnTickets];

template <typename V>
__device__ __forceinline__ void store_agent(V* p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V load_agent(const V* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Bit patterns in the order of the numbers, 0 below all; a NaN is below every number.
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  if (v != v) return 1;
  return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ unsigned long long lane_value(unsigned long long v, int lane) {
  const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t high = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return (unsigned long long)high << 32 | low;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  return __longlong_as_double((long long)lane_value((unsigned long long)__double_as_longlong(v), lane));
}

// A wave chooses a token's experts: the j-th is lane j's `expert`, with its logit; place[i] is what expert lane + 64 i is of
// them, 1 + j, or 0.  kMost logits a lane.
template <int kMost>
struct Choice {
  int expert, place[kMost];
  double logit[kMost], picked;
  __device__ __forceinline__ Choice(const W4MoeArgs& a, int t, unsigned long long* keys) : expert(0), picked(0.0) {
    const int lane = (int)threadIdx.x & 63, mine = (a.experts + 63) >> 6;
    const double* l = a.logits + (size_t)t * a.experts;
    uint32_t high[kMost], low[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const bool some = i < mine && lane + 64 * i < a.experts;
      logit[i] = some ? load_agent(l + lane + 64 * i) : 0.0;
      const unsigned long long key = some ? order_of(logit[i]) : 0;
      high[i] = (uint32_t)(key >> 32);
      low[i] = (uint32_t)key;
      place[i] = 0;
    }
    if constexpr (kMost == 1) {
      rank(a, (unsigned long long)high[0] << 32 | low[0], keys);
      return;
    }
#pragma unroll 1
    for (int j = 0; j < a.top_k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        if (i < mine) best = max(best, high[i]);
      best = wave_max(best);
      // Upper halves mostly tell them apart; where they do not, the lower halves do, and then the lower expert wins.
      int found = 0, at = 0, of = 0;
      uint32_t below = 0;
#pragma unroll
      for (int i = kMost - 1; i >= 0; --i) {
        if (i >= mine) continue;
        const unsigned long long has = __ballot(high[i] == best && place[i] == 0);
        found += __builtin_popcountll(has);
        if (has != 0) at = __builtin_ctzll(has), of = i;
        if (high[i] == best && place[i] == 0) below = max(below, low[i]);
      }
      if (found > 1) {
        below = wave_max(below);
#pragma unroll
        for (int i = kMost - 1; i >= 0; --i) {
          const unsigned long long has = __ballot(i < mine && high[i] == best && low[i] == below && place[i] == 0);
          if (has != 0) at = __builtin_ctzll(has), of = i;
        }
      }
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        if (i != of) continue;
        const double v = lane_value(logit[i], at);
        if (lane == j) picked = v, expert = at + 64 * i;
        if (lane == at) high[i] = low[i] = 0, place[i] = j + 1;
      }
    }
  }
  // Up to 64 experts: a lane counts the larger logits, read from LDS (a token's 8 of 64 0.6 us sooner than one after the
  // other).
  __device__ __forceinline__ void rank(const W4MoeArgs& a, unsigned long long key, unsigned long long* keys) {
    const int lane = (int)threadIdx.x & 63;
    keys[lane] = key;
    asm volatile("" ::: "memory");  // a wave's own words: its LDS operations stay in order
    int r = 0;
    for (int i = 0; i < a.experts; i += 16)
#pragma unroll
      for (int j = 0; j < 16; ++j) r += keys[i + j] > key ? 1 : 0;
    if (lane >= a.experts) r = lane;
    // Equal logits make equal ranks, whose sum is less than that of all: then the lower experts go first.
    int all = r;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
    if (all != 64 * 63 / 2)
      for (int i = 0; i < a.experts; ++i)
        if (keys[i] == key && i < lane && lane < a.experts) ++r;
    place[0] = lane < a.experts && r < a.top_k ? r + 1 : 0;
    expert = __builtin_amdgcn_ds_permute(4 * r, lane);
    const unsigned long long bits = (unsigned long long)__double_as_longlong(logit[0]);
    const uint32_t low = (uint32_t)__builtin_amdgcn_ds_permute(4 * r, (int)(uint32_t)bits);
    const uint32_t high = (uint32_t)__builtin_amdgcn_ds_permute(4 * r, (int)(uint32_t)(bits >> 32));
    picked = __longlong_as_double((long long)((unsigned long long)high << 32 | low));
  }
  // Leaves token t's experts and weights for the kernels that follow, and for the caller.
  __device__ __forceinline__ void leave(const W4MoeArgs& a, int t) const {
    const int lane = (int)threadIdx.x & 63, mine = (a.experts + 63) >> 6;
    const double top = lane_value(picked, 0), p = lane < a.top_k ? exp(picked - top) : 0.0;
    double sum = a.renormalise ? p : 0.0;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine && lane + 64 * i < a.experts) {
        if (!a.renormalise)
          sum += exp(logit[i] - top);
        else if (logit[i] != logit[i])
          sum = logit[i];  // the softmax over all experts has no value then
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
    if (a.tokens <= kMoeFewTokens)
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        if (i < mine && lane + 64 * i < a.experts)
          a.places[(size_t)t * a.experts + lane + 64 * i] = (uint8_t)place[i];
  }
};

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

// grid.x: four experts each, a wave one; grid.y: blocks of kTokens tokens (behind the last, the last one again).
template <typename T, int kMost, int kTokens>
__global__ __launch_bounds__(256) void moe_router_kernel(const W4MoeArgs a) {
  __shared__ int count[kMoeMaxExperts], start[kMoeMaxExperts], wave_sums[2][4];
  __shared__ unsigned long long keys[4][64];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int e = (int)blockIdx.x * 4 + wave, hidden = a.gate.k;
  const int first = (int)blockIdx.y * kTokens, tokens = min(a.tokens - first, kTokens);
  if (e < a.experts) {
    const float* w = a.router + (size_t)e * hidden;
    const T* x[kTokens];
    double sum[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      x[t] = static_cast<const T*>(a.x) + (size_t)(first + min(t, tokens - 1)) * a.x_stride;
      sum[t] = 0.0;
    }
    // Four columns a lane; the next eight (kTokens 1) or four steps' are on their way together.
    constexpr int kAhead = kTokens == 1 ? 8 : 4;
    int c = 4 * lane;
    for (; c + 256 * (kAhead - 1) + 4 <= hidden; c += 256 * kAhead) {
      float v[kAhead][4], u[kAhead][kTokens][4];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        load4(w + c + 256 * i, v[i]);
#pragma unroll
        for (int t = 0; t < kTokens; ++t) load4(x[t] + c + 256 * i, u[i][t]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[t] = __builtin_fma((double)u[i][t][j], (double)v[i][j], sum[t]);
    }
    for (; c < hidden; c += 256)
      for (int j = c; j < min(c + 4, hidden); ++j) {
        const double v = (double)w[j];
#pragma unroll
        for (int t = 0; t < kTokens; ++t) sum[t] = __builtin_fma((double)value(x[t] + j), v, sum[t]);
      }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const double s = wave_sum(sum[t]);
      if (lane == 0 && t < tokens) store_agent(a.logits + (size_t)(first + t) * a.experts + e, s);
    }
  }
  if (!last_to_arrive(&moe_tickets[1 + blockIdx.y], gridDim.x, &ticket)) return;
  if (wave < tokens) Choice<kMost>(a, first + wave, keys[wave]).leave(a, first + wave);
  if (a.tokens <= kMoeFewTokens) return;
  if (!last_to_arrive(&moe_tickets[0], gridDim.y, &ticket)) return;
  list_pairs(a, count, start, wave_sums);
}

// ------------------------------------------------------------------ the experts
// A reached expert and its pairs as a wave sees them.  Few tokens: lane t looks up whether token t chose the expert, and
// the rows' pairs go to the wave's own `list`; slot s is expert s, or where there are fewer pairs than experts that of pair
// s, unless an earlier token has it too.  More tokens: slot s of the lists.
struct Reached {
  int expert, count;
  const int32_t* pairs;
  template <bool kFew>
  __device__ __forceinline__ static Reached find(const W4MoeArgs& a, int slot, int32_t* list) {
    if constexpr (!kFew) {
      const MoeExpert ex = a.reached[slot];
      return Reached{ex.expert, ex.count, a.pairs + ex.start};
    }
    const int lane = (int)threadIdx.x & 63;
    const bool by_pair = a.tokens * a.top_k < a.experts;
    const int expert = __builtin_amdgcn_readfirstlane(by_pair ? a.chosen[slot] : slot);
    const int place = lane < a.tokens ? a.places[(size_t)lane * a.experts + expert] : 0;
    const unsigned long long has = __ballot(place != 0);
    if (by_pair && (has & ((1ull << (slot / a.top_k)) - 1)) != 0) return Reached{expert, 0, list};
    if (place != 0) list[__popcll(has & ((1ull << lane) - 1))] = lane * a.top_k + place - 1;
    asm volatile("" ::: "memory");  // a wave's own list: its LDS operations stay in order
    return Reached{expert, (int)__popcll(has), list};
  }
};

// Hidden columns 16 kTiles blockIdx.x .. of slot blockIdx.y: gate and up sums, the activation, terms.
template <typename T, int kSteps, W4Edge kEdge, int kTiles, int kWaves, bool kFew>
__global__ __launch_bounds__(64 * kWaves) void moe_hidden_kernel(const W4MoeArgs a) {
  typedef typename Kind<T>::Rows X;
  __shared__ float sums[kWaves][2 * kTiles][4][64];
  __shared__ int32_t lists[kFew ? kWaves : 1][kFew ? kMoeFewTokens : 1];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Reached ex = Reached::find<kFew>(a, (int)blockIdx.y, lists[kFew ? wave : 0]);
  if (16 * (int)blockIdx.z >= ex.count) return;
  const int tiles_k = a.gate.tiles_k;
  const u32x4* codes[2 * kTiles];
  const uint16_t* steps[2 * kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int tile = min((int)blockIdx.x * kTiles + i, a.gate.tiles_n - 1);
    codes[2 * i] = w4_codes(a.gate, ex.expert, tile);
    codes[2 * i + 1] = w4_codes(a.up, ex.expert, tile);
    steps[2 * i] = w4_steps<kSteps>(a.gate, ex.expert, tile);
    steps[2 * i + 1] = w4_steps<kSteps>(a.up, ex.expert, tile);
  }
  for (int block = 16 * (int)blockIdx.z; block < ex.count; block += 16 * (int)gridDim.z) {
    W4Tile<kSteps, 2 * kTiles> first;
    first.fetch(codes, steps, min(wave, tiles_k - 1));
    const int rows = min(ex.count - block, 16);
    const int mine = ex.pairs[block + min(lane & 15, rows - 1)];
    X x[1];
    x[0].p = static_cast<const T*>(a.x) + (size_t)((unsigned)mine / (unsigned)a.top_k) * a.x_stride;
    floatx4 acc[1][2 * kTiles] = {};
    w4_accumulate<kSteps, 2 * kTiles, 1, kEdge>(codes, steps, first, x, wave, tiles_k, kWaves, a.gate.k, acc);
    if (block >= 16 * (int)gridDim.z) __syncthreads();  // the sums before are read
#pragma unroll
    for (int i = 0; i < 2 * kTiles; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][i][r][lane] = acc[0][i][r];
    __syncthreads();
    for (int at = (int)threadIdx.x; at < rows * 16 * kTiles; at += 64 * kWaves) {
      const int row = at / (16 * kTiles), c = at % (16 * kTiles), i = c >> 4;
      const int r = row & 3, l = 16 * (row >> 2) + (c & 15);
      float g = sums[0][2 * i][r][l], u = sums[0][2 * i + 1][r][l];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) g += sums[w][2 * i][r][l], u += sums[w][2 * i + 1][r][l];
      const uint32_t f = blockIdx.x * (16 * kTiles) + (uint32_t)c;
      uint16_t* to = a.hidden + (size_t)ex.pairs[block + row] * a.hidden_stride;
      // Columns behind the last are zeros: whole tiles are multiplied.
      const float h = f < (uint32_t)a.gate.n ? activation(g, a.activation) * u : 0.0f;
      if (f < a.hidden_stride) put_terms(to + f, a.hidden_plane, h);
      if (blockIdx.x == gridDim.x - 1)
        for (uint32_t z = f + 16 * kTiles; z < a.hidden_stride; z += 16 * kTiles)
          put_terms(to + z, a.hidden_plane, 0.0f);
    }
  }
}

// The pairs' sums of a column group by token, weighed, in the order of the token's experts: items `first`, first + step ..
// of two columns.  kItems times kSums loads are on their way together: they come from behind the L2 caches.
template <typename T, int kColumns, int kItems, int kSums>
__device__ __forceinline__ void join_some(const W4MoeArgs& a, const float* sums, int column0, int first, int step) {
  constexpr int kTwos = kColumns / 2;
  const int items = a.tokens * kTwos, parts = a.top_k * a.parts;
  for (int at0 = first; at0 < items; at0 += kItems * step) {
    float v[kItems] = {}, u[kItems] = {};
    for (int q0 = 0; q0 < parts; q0 += kSums) {
      unsigned long long both[kItems][kSums];
      float w[kItems][kSums];
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int at = min(at0 + i * step, items - 1), token = at / kTwos;
#pragma unroll
        for (int q = 0; q < kSums; ++q) {
          const int part = min(q0 + q, parts - 1);
          both[i][q] = load_agent(reinterpret_cast<const unsigned long long*>(
              sums + ((size_t)token * parts + part) * kColumns + 2 * (at - token * kTwos)));
          w[i][q] = a.weights[token * a.top_k + part / a.parts];
        }
      }
#pragma unroll
      for (int i = 0; i < kItems; ++i)
#pragma unroll
        for (int q = 0; q < kSums; ++q)
          if (q0 + q < parts) {
            v[i] = __builtin_fmaf(w[i][q], __uint_as_float((uint32_t)both[i][q]), v[i]);
            u[i] = __builtin_fmaf(w[i][q], __uint_as_float((uint32_t)(both[i][q] >> 32)), u[i]);
          }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int at = at0 + i * step, token = at / kTwos, c = column0 + 2 * (at - token * kTwos);
      if (at >= items) break;
      T* to = static_cast<T*>(a.out) + (size_t)token * a.out_stride + c;
      if (c < a.down.n) put(to, v[i]);
      if (c + 1 < a.down.n) put(to + 1, u[i]);
    }
  }
}
template <typename T, int kColumns>
__device__ __forceinline__ void join(const W4MoeArgs& a, const float* sums, int column0, int first, int step) {
  if (a.top_k * a.parts <= 8)
    join_some<T, kColumns, 4, 8>(a, sums, column0, first, step);
  else
    join_some<T, kColumns, 1, 32>(a, sums, column0, first, step);
}

// Output columns 16 kNT blockIdx.x .. .  A unit is a part of K of a slot, a wave's; it leaves its sums by pair.  Where
// parts of K have a block of pairs at most (kParts), the slot's waves, neighbours in a workgroup, join their sums first.
// Few tokens: the last workgroup of a column group joins the pairs' sums.
template <typename T, int kSteps, int kNT, bool kFew, bool kParts>
__global__ __launch_bounds__(64 * kOutWaves) void moe_out_kernel(const W4MoeArgs a) {
  typedef W4RowsTerms<kHiddenTerms> X;
  constexpr int kColumns = 16 * kNT;
  __shared__ int32_t lists[kFew ? kOutWaves : 1][kFew ? kMoeFewTokens : 1];
  __shared__ float others[kParts ? kOutWaves : 1][kNT][4][64];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tiles_k = a.down.tiles_k, pairs = a.tokens * a.top_k, units = min(a.experts, pairs) * a.split;
  const int unit = (int)blockIdx.y * kOutWaves + wave, slot = unit / a.split, part = unit - slot * a.split;
  float* const sums = a.part + (size_t)blockIdx.x * pairs * a.parts * kColumns;  // [pair][part][kColumns]
  floatx4 acc[1][kNT];
  int mine = 0, rows = 0;
  const auto leave = [&](int at) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // Row 4 (lane / 16) + r: its pair is with the lane of that number.
      const int row = 4 * (lane >> 4) + r;
      float* const to = sums + ((size_t)__shfl(mine, row) * a.parts + at) * kColumns + (lane & 15);
      if (row < rows)
#pragma unroll
        for (int i = 0; i < kNT; ++i) store_agent(to + 16 * i, acc[0][i][r]);
    }
  };
  if (unit < units) {
    const Reached ex = Reached::find<kFew>(a, slot, lists[kFew ? wave : 0]);
    const int begin = tiles_k * part / a.split, end = tiles_k * (part + 1) / a.split;
    const u32x4* codes[kNT];
    const uint16_t* steps[kNT];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      const int tile = min((int)blockIdx.x * kNT + i, a.down.tiles_n - 1);
      codes[i] = w4_codes(a.down, ex.expert, tile);
      steps[i] = w4_steps<kSteps>(a.down, ex.expert, tile);
    }
    for (int block = 16 * (int)blockIdx.z; block < ex.count; block += 16 * (int)gridDim.z) {
      W4Tile<kSteps, kNT> first;
      first.fetch(codes, steps, begin);
      rows = min(ex.count - block, 16);
      mine = ex.pairs[block + min(lane & 15, rows - 1)];
      X x[1];
      x[0].plane = a.hidden_plane;
      x[0].p = a.hidden + (size_t)mine * a.hidden_stride;
#pragma unroll
      for (int i = 0; i < kNT; ++i) acc[0][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      w4_accumulate<kSteps, kNT, 1, kEdgeNone>(codes, steps, first, x, begin, end, 1, a.down.k, acc);
      if constexpr (!kParts) leave(part);
    }
  }
  if constexpr (kParts) {
    if (part > 0 && rows > 0)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) others[wave][i][r][lane] = acc[0][i][r];
    __syncthreads();
    if (part == 0 && rows > 0) {
      for (int p = 1; p < a.split; ++p)
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[0][i][r] += others[wave + p][i][r][lane];
      leave(0);
    }
  }
  if constexpr (kFew) {
    if (!a.joins || !last_to_arrive(&moe_column_tickets[blockIdx.x], gridDim.y, &ticket)) return;
    join<T, kColumns>(a, sums, (int)blockIdx.x * kColumns, (int)threadIdx.x, 64 * kOutWaves);
  }
}

// Column groups blockIdx.x, and blockIdx.y's share of their tokens.
template <typename T, int kNT>
__global__ __launch_bounds__(256) void moe_join_kernel(const W4MoeArgs a) {
  constexpr int kColumns = 16 * kNT;
  join<T, kColumns>(a, a.part + (size_t)blockIdx.x * a.tokens * a.top_k * a.parts * kColumns, (int)blockIdx.x * kColumns,
                    (int)(blockIdx.y * 256 + threadIdx.x), (int)gridDim.y * 256);
}

template <typename T, int kSteps, W4Edge kEdge>
hipError_t launch_hidden(const W4MoeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.gate.tiles_n + kHiddenTiles - 1) / kHiddenTiles,
                  (unsigned)std::min(a.experts, a.tokens * a.top_k), (unsigned)a.blocks);
#define HIDDEN(FEW)                                                                                                       \
  hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kEdge, kHiddenTiles, kHiddenWaves, FEW>), grid, dim3(64 * kHiddenWaves), \
                     0, stream, a)
  if (a.tokens <= kMoeFewTokens)
    HIDDEN(true);
  else
    HIDDEN(false);
#undef HIDDEN
  return hipGetLastError();
}
template <typename T, int kSteps>
hipError_t launch_hidden(const W4MoeArgs& a, hipStream_t stream) {
  const W4Edge edge = w4_edge<T>(a.x, a.x_stride, a.gate.k);
  if (edge == kEdgeNone) return launch_hidden<T, kSteps, kEdgeNone>(a, stream);
  if (edge == kEdgeShift) return launch_hidden<T, kSteps, kEdgeShift>(a, stream);
  if constexpr (sizeof(T) == 2)
    if (edge == kEdgeOdd) return launch_hidden<T, kSteps, kEdgeOdd>(a, stream);
  return launch_hidden<T, kSteps, kEdgeShort>(a, stream);
}

template <typename T, int kSteps, int kNT, bool kFew, bool kParts>
hipError_t launch_out(const W4MoeArgs& a, hipStream_t stream) {
  const unsigned columns = (unsigned)(a.down.tiles_n + kNT - 1) / kNT;
  const unsigned units = (unsigned)(std::min(a.experts, a.tokens * a.top_k) * a.split);
  const dim3 grid(columns, (units + kOutWaves - 1) / kOutWaves, (unsigned)a.blocks);
  hipLaunchKernelGGL((moe_out_kernel<T, kSteps, kNT, kFew, kParts>), grid, dim3(64 * kOutWaves), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.joins) return e;
  const unsigned shares = (unsigned)std::min((a.tokens * 8 * kNT + 255) / 256, 64);
  hipLaunchKernelGGL((moe_join_kernel<T, kNT>), dim3(columns, shares), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <typename T, int kSteps>
hipError_t launch_out(const W4MoeArgs& a, hipStream_t stream) {
  if (a.tokens <= kMoeFewTokens) {
    if (a.out_tiles == 4) return launch_out<T, kSteps, 4, true, false>(a, stream);
    if (a.split > a.parts) return launch_out<T, kSteps, 2, true, true>(a, stream);
    return launch_out<T, kSteps, 2, true, false>(a, stream);
  }
  if (a.out_tiles == 4) return launch_out<T, kSteps, 4, false, false>(a, stream);
  return launch_out<T, kSteps, 2, false, false>(a, stream);
}

template <typename T>
hipError_t launch(const W4MoeArgs& a, hipStream_t stream) {
  const dim3 router((unsigned)(a.experts + 3) / 4, (unsigned)(a.tokens + kTokenBlock - 1) / kTokenBlock);
#define ROUTER(MOST)                                                                                  \
  if (a.tokens == 1)                                                                                  \
    hipLaunchKernelGGL((moe_router_kernel<T, MOST, 1>), router, dim3(256), 0, stream, a);             \
  else                                                                                                \
    hipLaunchKernelGGL((moe_router_kernel<T, MOST, kTokenBlock>), router, dim3(256), 0, stream, a);
  if (a.experts <= 64) {
    ROUTER(1)
  } else if (a.experts <= 256) {
    ROUTER(4)
  } else {
    ROUTER(16)
  }
#undef ROUTER
  // What reads a launch's results is queued only behind one that is.
  hipError_t e = hipGetLastError();
#define STEPS(what, group)                    \
  if (e == hipSuccess)                        \
    e = group == 32   ? what<T, 4>(a, stream) \
        : group == 64 ? what<T, 2>(a, stream) \
                      : what<T, 1>(a, stream);
  STEPS(launch_hidden, a.gate.group)
  STEPS(launch_out, a.down.group)
#undef STEPS
  return e;
}

}  // namespace

size_t moe_w4_workspace(W4MoeArgs& a, void* base) {
  const size_t pairs = (size_t)a.tokens * a.top_k, experts = (size_t)a.experts;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* p = static_cast<char*>(base) + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  // Few slots: K is dealt out too.  Many: more columns a workgroup, which share the hidden rows (64 experts of 1024 hidden
  // and 2048 outer columns: 32 slots 13.7 us with 32 columns, 16.5 with 64; 64 slots of 8 tokens 21 and 18, of 64 tokens 42
  // and 30).
  const int slots = (int)std::min(experts, pairs);
  a.out_tiles = slots >= 64 ? 4 : 2;
  const int columns = (a.down.tiles_n + a.out_tiles - 1) / a.out_tiles;
  a.split = 1;
  while (a.split < 4 && slots * a.split < 32 && a.down.tiles_k >= 4 * a.split) a.split *= 2;
  a.parts = a.tokens <= 16 ? 1 : a.split;
  a.joins = a.tokens <= kMoeFewTokens && columns <= kColumnTickets;
  // Blocks of sixteen pairs of an expert at once, for twice as many pairs as experts have in the mean; those behind are taken
  // in turn.
  a.blocks = a.tokens <= kMoeFewTokens ? 1 : (int)std::min<size_t>(std::max<size_t>(2 * pairs / experts + 15, 16) / 16, 64);
  a.hidden_stride = (uint32_t)a.down.tiles_k * kW4TileK;
  a.hidden_plane = pairs * a.hidden_stride;
  a.logits = reinterpret_cast<double*>(take((size_t)a.tokens * experts * sizeof(double)));
  a.chosen = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.weights = reinterpret_cast<float*>(take(pairs * sizeof(float)));
  a.places = reinterpret_cast<uint8_t*>(take((size_t)a.tokens * experts));
  a.pairs = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.reached = reinterpret_cast<MoeExpert*>(take((size_t)slots * sizeof(MoeExpert)));
  a.hidden = reinterpret_cast<uint16_t*>(take(a.hidden_plane * kHiddenTerms * sizeof(uint16_t)));
  const size_t parts = pairs * a.parts * columns * 16u * a.out_tiles;
  a.part = reinterpret_cast<float*>(take(parts * sizeof(float)));
  return at;
}

hipError_t launch_moe_w4(const W4MoeArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<uint16_t>(a, stream) : launch<float>(a, stream);
}

}  // namespace prom
