// A mixture-of-experts layer of a few tokens on 4-bit weights:
//   l = x router^T, a token's experts the top_k largest l (ties to the lower expert), p their softmax weights,
//   out = sum_e p_e (act(x gate_e^T) * (x up_e^T)) down_e^T.
//
// Three launches.  The router: a wave makes an expert's logits of four tokens, in binary64 (a choice between two close
// experts does not depend on the order of a sum); the last workgroup of four tokens' (tickets.h) chooses their experts, and
// the last of those lists the pairs, a token with one of its experts, by expert.  The hidden columns: a workgroup takes 16
// of one reached expert, its gate and up weights once for sixteen pairs at a time (w4_product.h), and leaves the hidden
// rows as bf16 terms, in the form that the second product multiplies.  The output columns: a workgroup takes 16 of all
// experts, its waves an expert (or a part of its K) each, weighs their sums and adds them by token in LDS.  Above 64 tokens
// the products' sums by pair go to memory and are joined in a fourth launch.
//
// Bound by the reached experts' weights, and for a token by the latency of three kernels that follow one another.  64
// experts of 1024 with 2048 outer columns, 8 a token, in bf16: a token 6.4 + 6.0 + 6.6 us (28 MB at 2.2 TB/s in the last two), 64
// tokens, which reach all experts, 10.2 + 33.5 + 28.5 us (214 MB at 3.5 TB/s; 64 rows of x and of the hidden columns come from L2
// for each workgroup).
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
constexpr int kColumnTickets = 256, kMaxSlices = 8;
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

// A wave chooses token t's experts, one after the other, and makes their weights; kMost logits a lane.
template <int kMost>
__device__ __forceinline__ void choose(const W4MoeArgs& a, int t) {
  const int lane = (int)threadIdx.x & 63;
  const double* l = a.logits + (size_t)t * a.experts;
  const int mine = (a.experts + 63) >> 6;
  double logit[kMost];
  unsigned long long key[kMost];
  int place[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    key[i] = 0;
    place[i] = 0;
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
      if (lane == at) key[i] = 0, place[i] = j + 1;
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
  if (a.tokens <= kMoeFewTokens)
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine && lane + 64 * i < a.experts)
        a.places[(size_t)t * a.experts + lane + 64 * i] = (uint8_t)place[i];
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

// grid.x: four experts each, a wave one; grid.y: blocks of kTokens tokens (behind the last, the last one again).
template <typename T, int kMost, int kTokens>
__global__ __launch_bounds__(256) void moe_router_kernel(const W4MoeArgs a) {
  __shared__ int count[kMoeMaxExperts], start[kMoeMaxExperts], wave_sums[2][4];
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
  if (wave < tokens) choose<kMost>(a, first + wave);
  if (a.tokens <= kMoeFewTokens) return;
  if (!last_to_arrive(&moe_tickets[0], gridDim.y, &ticket)) return;
  list_pairs(a, count, start, wave_sums);
}

// ------------------------------------------------------------------ the experts
// A reached expert and its pairs as a wave sees them.  Few tokens: lane t looks up whether token t chose the expert, and the
// rows' pairs go to the wave's own `list`; slot s is expert s, or where there are fewer pairs than experts that of pair s, unless
// an earlier token has it too.  More tokens: slot s of the lists.
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
  if (ex.count == 0) return;
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
  for (int block = 0; block < ex.count; block += 16) {
    W4Tile<kSteps, 2 * kTiles> first;
    first.fetch(codes, steps, min(wave, tiles_k - 1));
    const int rows = min(ex.count - block, 16);
    const int mine = ex.pairs[block + min(lane & 15, rows - 1)];
    X x[1];
    x[0].p = static_cast<const T*>(a.x) + (size_t)((unsigned)mine / (unsigned)a.top_k) * a.x_stride;
    floatx4 acc[1][2 * kTiles] = {};
    w4_accumulate<kSteps, 2 * kTiles, 1, kEdge>(codes, steps, first, x, wave, tiles_k, kWaves, a.gate.k, acc);
    if (block > 0) __syncthreads();  // the sums before are read
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
      if (f < a.hidden_stride) put_terms(to + f, a.hidden_plane, h, T());
      if (blockIdx.x == gridDim.x - 1)
        for (uint32_t z = f + 16 * kTiles; z < a.hidden_stride; z += 16 * kTiles)
          put_terms(to + z, a.hidden_plane, 0.0f, T());
    }
  }
}

// Few tokens: output columns 16 kNT blockIdx.x .. .  A unit is a part of K of a slot; those of slice blockIdx.y are dealt to
// the waves, which weigh their sums and add them by token in LDS, each in its own place.
template <typename T, int kSteps, int kNT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void moe_out_kernel(const W4MoeArgs a) {
  typedef W4RowsTerms<Kind<T>::kHiddenTerms> X;
  constexpr int kColumns = 16 * kNT, kPart = kMoeFewTokens * kColumns;
  extern __shared__ float sums[];  // [kWaves][tokens][kColumns]
  __shared__ int32_t lists[kWaves][kMoeFewTokens];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tiles_k = a.down.tiles_k, slots = min(a.experts, a.tokens * a.top_k);
  const int count = a.tokens * kColumns;
  float* own = sums + wave * count;
  for (int at = lane; at < count; at += 64) own[at] = 0.0f;
  for (int unit = (int)blockIdx.y * kWaves + wave; unit < slots * a.split; unit += kWaves * a.slices) {
    const int slot = unit / a.split, part = unit - slot * a.split;
    const Reached ex = Reached::find<true>(a, slot, lists[wave]);
    const int begin = tiles_k * part / a.split, end = tiles_k * (part + 1) / a.split;
    if (ex.count == 0 || begin == end) continue;
    const u32x4* codes[kNT];
    const uint16_t* steps[kNT];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      const int tile = min((int)blockIdx.x * kNT + i, a.down.tiles_n - 1);
      codes[i] = w4_codes(a.down, ex.expert, tile);
      steps[i] = w4_steps<kSteps>(a.down, ex.expert, tile);
    }
    for (int block = 0; block < ex.count; block += 16) {
      W4Tile<kSteps, kNT> first;
      first.fetch(codes, steps, begin);
      const int rows = min(ex.count - block, 16);
      const int mine = ex.pairs[block + min(lane & 15, rows - 1)];
      const float weight = a.weights[mine];
      X x[1];
      x[0].plane = a.hidden_plane;
      x[0].p = a.hidden + (size_t)mine * a.hidden_stride;
      floatx4 acc[1][kNT] = {};
      w4_accumulate<kSteps, kNT, 1, kEdgeNone>(codes, steps, first, x, begin, end, 1, a.down.k, acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // Row 4 (lane / 16) + r: its pair and weight are with the lane of that number.  An expert's rows are of different
        // tokens.
        const int row = 4 * (lane >> 4) + r;
        const int token = (int)((unsigned)__shfl(mine, row) / (unsigned)a.top_k);
        const float p = __shfl(weight, row);
        if (row < rows)
#pragma unroll
          for (int i = 0; i < kNT; ++i) own[token * kColumns + 16 * i + (lane & 15)] += p * acc[0][i][r];
      }
    }
  }
  __syncthreads();
  const int column0 = (int)blockIdx.x * kColumns;
  T* out = static_cast<T*>(a.out) + column0;
  float* part = a.part + (size_t)blockIdx.x * a.slices * kPart;
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    float v = sums[at];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w * count + at];
    if (a.slices > 1)
      store_agent(part + (size_t)blockIdx.y * kPart + at, v);
    else if (column0 + at % kColumns < a.down.n)
      put(out + (size_t)(at / kColumns) * a.out_stride + at % kColumns, v);
  }
  if (a.slices == 1 || !last_to_arrive(&moe_column_tickets[blockIdx.x], (uint32_t)a.slices, &ticket)) return;
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    float p[kMaxSlices];
#pragma unroll
    for (int s = 0; s < kMaxSlices; ++s) p[s] = s < a.slices ? load_agent(part + (size_t)s * kPart + at) : 0.0f;
    float v = p[0];
#pragma unroll
    for (int s = 1; s < kMaxSlices; ++s) v += p[s];
    if (column0 + at % kColumns < a.down.n) put(out + (size_t)(at / kColumns) * a.out_stride + at % kColumns, v);
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

template <typename T, int kSteps, W4Edge kEdge>
void launch_hidden(const W4MoeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.gate.tiles_n + kHiddenTiles - 1) / kHiddenTiles,
                  (unsigned)std::min(a.experts, a.tokens * a.top_k));
#define HIDDEN(FEW)                                                                                                       \
  hipLaunchKernelGGL((moe_hidden_kernel<T, kSteps, kEdge, kHiddenTiles, kHiddenWaves, FEW>), grid, dim3(64 * kHiddenWaves), \
                     0, stream, a)
  if (a.tokens <= kMoeFewTokens)
    HIDDEN(true);
  else
    HIDDEN(false);
#undef HIDDEN
}
template <typename T, int kSteps>
void launch_hidden(const W4MoeArgs& a, hipStream_t stream) {
  if (a.gate.k % kW4TileK == 0)
    launch_hidden<T, kSteps, kEdgeNone>(a, stream);
  else if (a.gate.k >= 8)
    launch_hidden<T, kSteps, kEdgeShift>(a, stream);
  else
    launch_hidden<T, kSteps, kEdgeShort>(a, stream);
}

template <typename T, int kSteps>
void launch_out(const W4MoeArgs& a, hipStream_t stream) {
  if (a.tokens <= kMoeFewTokens) {
    const dim3 grid((unsigned)(a.down.tiles_n + a.out_tiles - 1) / (unsigned)a.out_tiles, (unsigned)a.slices);
    const unsigned lds = kOutWaves * (unsigned)a.tokens * 16u * (unsigned)a.out_tiles * sizeof(float);
    if (a.out_tiles == 2)
      hipLaunchKernelGGL((moe_out_kernel<T, kSteps, 2, kOutWaves>), grid, dim3(64 * kOutWaves), lds, stream, a);
    else
      hipLaunchKernelGGL((moe_out_kernel<T, kSteps, 4, kOutWaves>), grid, dim3(64 * kOutWaves), lds, stream, a);
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
  // Few slots: K is dealt out too.  Many: more columns a workgroup, which share the hidden rows (64 experts of 1024 hidden
  // and 2048 output columns, 32 slots 11.9 us with 32 columns, 14.6 with 64; 64 slots of 8 tokens 18 to 21 and 15.7, of 64
  // tokens 33 to 38 and 28.7).
  const int slots = (int)std::min(experts, pairs);
  a.out_tiles = slots >= 64 ? 4 : 2;
  const int columns = (a.down.tiles_n + a.out_tiles - 1) / a.out_tiles;
  a.split = 1;
  a.slices = 1;
  while (a.split < 4 && slots * a.split < 32 && a.down.tiles_k >= 4 * a.split) a.split *= 2;
  while (a.slices < kMaxSlices && columns * a.slices < 256 && slots * a.split >= 2 * kOutWaves * a.slices) a.slices *= 2;
  a.hidden_stride = (uint32_t)a.down.tiles_k * kW4TileK;
  a.hidden_plane = pairs * a.hidden_stride;
  a.logits = reinterpret_cast<double*>(take((size_t)a.tokens * experts * sizeof(double)));
  a.chosen = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.weights = reinterpret_cast<float*>(take(pairs * sizeof(float)));
  a.places = reinterpret_cast<uint8_t*>(take((size_t)a.tokens * experts));
  a.pairs = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
  a.reached = reinterpret_cast<MoeExpert*>(take((size_t)slots * sizeof(MoeExpert)));
  a.hidden = reinterpret_cast<uint16_t*>(take(a.hidden_plane * (bf16 ? 2 : 3) * sizeof(uint16_t)));
  const size_t parts = a.tokens <= kMoeFewTokens ? (size_t)columns * a.slices * (kMoeFewTokens * 16u * (unsigned)a.out_tiles)
                                                 : pairs * (size_t)a.down.n;
  a.part = reinterpret_cast<float*>(take(parts * sizeof(float)));
  return at;
}

hipError_t launch_moe_w4(const W4MoeArgs& a, bool bf16, hipStream_t stream) {
  return bf16 ? launch<uint16_t>(a, stream) : launch<float>(a, stream);
}

}  // namespace prom
