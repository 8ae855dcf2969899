// Attention over the 4-bit paged cache (kv4_cache.hip):
// o[r, h] = sum_t softmax_t(scale q[r, h] . k[t]) v[t], k[t] = s code, v[t] = s code
// with a step s for 64 channels of a token's head.
//
// Rows are (row, query head of the group) pairs: a tile is 16 of them, so that the heads
// that share a key head, and a few rows of a prompt, read the cache once.  A wave takes
// a page (64 tokens) at a time:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16.  E2M1 codes are exact in bf16 (one
//   instruction turns two codes into two numbers), so K goes into the products as codes,
//   one accumulator a group of 64 channels, and the groups' steps are applied to the
//   scores in fp32.  A lane owns one row and 16 of the page's scores: tile c, register i
//   of lane (h, row) is token 16 h + 4 c + i, so a lane's tokens are neighbours and their
//   steps four 16-byte loads.
//   Softmax with a running maximum that follows only when it grew by more than 2^8, in
//   base 2.
//   O^T = V^T P^T.  V's step goes to the probability; P s is split into bf16 terms
//   that carry it to 16 bits (24 for fp32 rows), the codes again are exact.  The V^T
//   operand (16 channels, tokens in k) comes from ds_read_b64_tr_b4, which hands a lane
//   the 16 tokens of its channel; S^T's register order is already P^T's operand order.
//   fp32 queries are three bf16 terms (exact).
// No rounding but P's and fp32's is made anywhere.
//
// Pages of a sequence are dealt to the waves of a workgroup and to gridDim splits; the
// waves join through LDS, splits through fp32 partials and a second kernel, in a fixed
// order.  Bound by reading the cache for long sequences (272 bytes of a 64-channel
// group pair... per token and head D + D / 16 bytes).
#include <algorithm>

#include "reactor_internal.h"

namespace prom {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

constexpr float kLazyLog2 = 8.0f;
constexpr int kTileRows = 16;
constexpr int kWaves = 4;
constexpr int kMaxSplits = 64;  // a lane each when they are joined
constexpr uint64_t kMostPartialBytes = 1ull << 30;

struct Kv4Kernel {
  Kv4View c;
  const void* q;
  void* out;
  const int32_t* starts;
  float* part;  // sums [splits][rows][q_heads][D], then (maximum, weight) [splits][rows][q_heads]
  size_t ends;  // where these begin
  int rows, q_stride, out_stride;
  int q_heads, group, tiles, splits;
  int split_shift;  // a split has 2^split_shift pages or a share of more
  int window;       // 0: none
  float scale_log2;
  uint32_t group_shift;
  uint64_t group_magic;

  // x / group for 0 <= x < 2^31: with 2^l >= group, floor(2^(31 + l) / group) + 1 is over the
  // quotient by at most 2^l / 2^(31 + l), which no such x carries past a whole number.
  __device__ __forceinline__ int over_group(int x) const {
    return (int)(((uint64_t)(uint32_t)x * group_magic) >> group_shift);
  }
};

typedef const __attribute__((address_space(4))) int32_t Constant;

// A sequence's rows (within the call's) and length.
struct Sequence {
  int first, n, length;
  __device__ __forceinline__ Sequence(const Kv4Kernel& g, int seq) {
    Constant* starts = (Constant*)g.starts;
    first = min(max(starts[seq], 0), g.rows);
    n = min(max(starts[seq + 1], 0), g.rows) - first;
    length = max(((Constant*)g.c.lengths)[seq], 0);
  }
};

// The positions of a tile's first and last row, the pages that they see between them, and into
// how many splits these are dealt.  Past the table every token is bad: the page behind its last
// stands for all of them.
struct Tile {
  int pos0, pos1, page0, last, splits;
  __device__ __forceinline__ Tile(const Kv4Kernel& g, const Sequence& s, int tile) {
    const int x0 = tile * kTileRows, from = s.length - s.n;
    pos0 = from + g.over_group(x0);
    pos1 = from + g.over_group(min(x0 + kTileRows, s.n * g.group) - 1);
    page0 = g.window && pos0 >= g.window ? min((pos0 - g.window + 1) / kKv4Page, g.c.table_stride) : 0;
    last = pos1 < 0 ? 0 : min(pos1 / kKv4Page, g.c.table_stride) + 1;
    splits = min(g.splits, max(1, (last - page0 + (1 << g.split_shift) - 1) >> g.split_shift));
  }
};

__device__ __forceinline__ float* ends(const Kv4Kernel& g) { return g.part + g.ends; }

// max / sum of v over lanes l and l ^ 16.
__device__ __forceinline__ float max_rows16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_rows16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The eight numbers of a word of codes.
__device__ __forceinline__ bf16x8 numbers(uint32_t codes) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Steps 2 j and 2 j + 1 of a word of two.
__device__ __forceinline__ float step_of(uint32_t w, int odd) {
  return __uint_as_float(odd ? w & 0xFFFF0000u : w << 16);
}

// kN bf16 terms that add up to x: each but the last is cut off (toward zero), so that the
// rest is exact; the last is rounded.
template <int kN>
__device__ __forceinline__ void terms(float x, __bf16 (&t)[kN]) {
#pragma unroll
  for (int i = 0; i + 1 < kN; ++i) {
    const uint32_t top = __float_as_uint(x) & 0xFFFF0000u;
    t[i] = __builtin_bit_cast(__bf16, (uint16_t)(top >> 16));
    x -= __uint_as_float(top);
  }
  t[kN - 1] = (__bf16)x;
}

// One head's part of a page in LDS, as it lies in memory but for the order of the 16-byte
// chunks within a token's row, which is chosen so that an operand read's 16 tokens fall into
// different banks: chunk c of token t is at c ^ key_swz(t) (tokens 16 a + 4 c + b for one c are
// read together) or c ^ value_swz(t) (16 neighbours).  Filled by whole transfers of 1 KiB.
template <int D>
struct Stage {
  static constexpr int kRow = D / 2;
  static constexpr int kCodes = kKv4Page * kRow;  // keys, then values
  static constexpr int kSteps = 2 * kCodes;       // keys' steps [D / 64][64], then the values'
  static constexpr int kMoves = (kv4_block_bytes(D) + 1023) / 1024;
  static constexpr int kBytes = 1024 * kMoves;
  static_assert(2 * kMoves < 64, "transfers in flight");

  __device__ static __forceinline__ int key_swz(int t) {
    return D == 64 ? (t >> 4) & 1 : D == 128 ? (t >> 4) & 3 : ((t >> 4) & 3) | ((t << 1) & 4);
  }
  __device__ static __forceinline__ int value_swz(int t) {
    return D == 64 ? (t >> 3) & 1 : D == 128 ? (t >> 2) & 3 : (t >> 1) & 7;
  }
  // Queues the transfers of a block to LDS address `to` (a wave's own stage).
  __device__ static __forceinline__ void fill(const uint8_t* block, uint32_t to, int lane) {
    const unsigned long long a = (unsigned long long)block;
    intx4 d;
    d.x = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffu));
    d.y = __builtin_amdgcn_readfirstlane((int)(a >> 32));
    d.z = kv4_block_bytes(D);
    d.w = 0x00020000;
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int at = 1024 * i + 16 * lane;
      uint32_t off = (uint32_t)at;
      if (1024 * i < kSteps) {
        const int t = at % kCodes / kRow;
        off ^= (uint32_t)(16 * (1024 * i < kCodes ? key_swz(t) : value_swz(t)));
      }
      const uint32_t m0 = __builtin_amdgcn_readfirstlane(to + 1024 * i);
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(m0), "v"(off), "s"(d)
                   : "memory", "m0");
    }
  }
};

template <bool kF32, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void kv4_attention_kernel(const Kv4Kernel g) {
  constexpr int kG = D / 64, kQT = kF32 ? 3 : 1, kPT = kF32 ? 3 : 2;
  constexpr int kSteps = D / 32;  // MFMA steps of 32 channels
  constexpr int kB = D / 16;      // blocks of 16 output channels
  using St = Stage<D>;
  constexpr int kJoinBytes = kTileRows * (D + 4) * 4;  // a wave's sums [16][D], maxima, weights
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * (2 * St::kBytes > kJoinBytes ? 2 * St::kBytes : kJoinBytes)];

  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r16 = lane & 15, h = lane >> 4;
  // Splits fastest, then key heads, then tiles, then sequences.
  uint32_t b = blockIdx.x;
  const int split = (int)(b % (uint32_t)g.splits);
  b /= (uint32_t)g.splits;
  const int head = (int)(b % (uint32_t)g.c.kv_heads);
  b /= (uint32_t)g.c.kv_heads;
  const int tile0 = (int)(b % (uint32_t)g.tiles);
  const int seq = (int)(b / (uint32_t)g.tiles);

  const Sequence sq(g, seq);
  if (sq.n <= 0) return;
  // Constant address space: page numbers come by scalar loads, which do not wait for the
  // transfers of pages as vector loads would.
  const auto* table = (const Constant*)(g.c.table + (size_t)seq * g.c.table_stride);
  const uint8_t* mine_lds = lds + wave * 2 * St::kBytes;
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) const uint8_t*)mine_lds;

  const int pairs = sq.n * g.group;
  for (int tile = tile0; tile * kTileRows < pairs; tile += g.tiles) {
    const Tile tl(g, sq, tile);
    if (split >= tl.splits) continue;
    // This lane's row: pair x = row * group + query head.  Lanes without one work on zeros.
    const int x0 = tile * kTileRows, x = x0 + r16;
    const bool mine = x < pairs;
    const int row = mine ? g.over_group(x) : 0;
    const int q_head = head * g.group + (mine ? x - row * g.group : 0);
    const int pos = mine ? sq.length - sq.n + row : tl.pos1;             // its position
    const int low = g.window && pos >= g.window ? pos - g.window : -1;  // it sees low < t <= pos
    const int page0 = tl.page0, last = tl.last;

    // Q^T operand: lane (h, row), step s: channels 32 s + 8 h .. + 7.
    bf16x8 q[kSteps][kQT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const size_t at = (size_t)(sq.first + row) * g.q_stride + (size_t)q_head * D + 32 * s + 8 * h;
      if constexpr (kF32) {
        float v[8];
        __builtin_memcpy(v, static_cast<const float*>(g.q) + at, 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          __bf16 t[kQT];
          terms(mine ? v[j] : 0.0f, t);
#pragma unroll
          for (int i = 0; i < kQT; ++i) q[s][i][j] = t[i];
        }
      } else {
        u32x4 v;
        __builtin_memcpy(&v, static_cast<const uint16_t*>(g.q) + at, 16);
        if (!mine) v = u32x4{0u, 0u, 0u, 0u};
        q[s][0] = __builtin_bit_cast(bf16x8, v);
      }
    }

    floatx4 o[kB] = {};
    float m_run = -INFINITY, m_log2 = 0.0f, l_run = 0.0f;

    const int stride = tl.splits * kWaves;
    int pg = page0 + split * kWaves + wave;
    auto page_number = [&](int p) -> uint32_t {
      return p < last && p < g.c.table_stride ? (uint32_t)table[p] : 0xFFFFFFFFu;
    };
    auto page_block = [&](uint32_t number) -> const uint8_t* {
      const uint32_t ok = number < g.c.pages ? number : 0u;
      return g.c.pool + ((size_t)ok * g.c.kv_heads + head) * kv4_block_bytes(D);
    };
    // Two stages: the next page is on its way while this one is worked on.  The transfers
    // are the loop's only vector memory operations, and a wave waits for its own alone.
    uint32_t number = page_number(pg), next_number = page_number(pg + stride);
    int now = 0;
    if (pg < last) St::fill(page_block(number), lds0, lane);
    for (; pg < last; pg += stride) {
      // The other stage's reads have returned before it is filled again.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const uint32_t after = page_number(pg + 2 * stride);
      if (pg + stride < last) {
        St::fill(page_block(next_number), lds0 + (now ^ 1) * St::kBytes, lane);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(St::kMoves) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const uint8_t* stage = mine_lds + now * St::kBytes;

      u32x4 ks[kG][2];
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          ks[gr][j] = *reinterpret_cast<const u32x4*>(stage + St::kSteps + 128 * gr + 32 * h + 16 * j);
      floatx4 s[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // Row r of the operand is token 16 (r / 4) + 4 c + r % 4.
        const int t = 16 * (r16 >> 2) + 4 * c + (r16 & 3);
        uint32_t k[kSteps];
        if constexpr (D == 64) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(stage + t * St::kRow + ((8 * h) ^ (16 * St::key_swz(t))));
          k[0] = w.x, k[1] = w.y;
        } else {
#pragma unroll
          for (int j = 0; j < kSteps / 4; ++j) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(stage + t * St::kRow + 16 * ((4 * j + h) ^ St::key_swz(t)));
            k[4 * j] = w.x, k[4 * j + 1] = w.y, k[4 * j + 2] = w.z, k[4 * j + 3] = w.w;
          }
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          floatx4 acc = {};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int st = 2 * gr + u;
            const bf16x8 kf = numbers(k[st]);
#pragma unroll
            for (int i = 0; i < kQT; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[st][i], acc, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 4 * c + i;
            const float step = step_of(ks[gr][j / 8][j / 2 % 4], j & 1);
            s[c][i] = gr == 0 ? acc[i] * step : __builtin_fmaf(acc[i], step, s[c][i]);
          }
        }
      }
      // Masked where the page has tokens that some row does not see, or is bad.
      const bool bad = number >= g.c.pages, past = pg >= g.c.table_stride;
      const int t0 = pg * kKv4Page;
      const bool edge = bad || t0 + (kKv4Page - 1) > tl.pos0 || (g.window && t0 <= tl.pos1 - g.window);
      uint32_t seen = 0;  // bit j: token 16 h + j
      if (edge) {
        // A row that lies past its table sees its own token at least, which is bad.
        const bool lost = past && pos / kKv4Page >= g.c.table_stride;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = t0 + 16 * h + 4 * c + i;
            const bool sees = past ? lost : t <= pos && t > low;
            if (bad) s[c][i] = NAN;
            if (!sees) s[c][i] = -INFINITY;
            seen |= (uint32_t)sees << (4 * c + i);
          }
      }
      float m = s[0][0];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, s[c][i]);
      m = max_halves(max_rows16(m));
      // (-inf) - (-inf) is NaN, which is not above: such a row has seen nothing yet.
      if (__any((m - m_run) * g.scale_log2 > kLazyLog2)) {
        const float m_new = fmaxf(m, m_run);
        const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f((m_run - m_new) * g.scale_log2);
        m_run = m_new;
        m_log2 = m_new == -INFINITY ? 0.0f : m_new * g.scale_log2;
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < kB; ++i) o[i] *= alpha;
      }
      float p[16];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][i], g.scale_log2, -m_log2));
          p[4 * c + i] = e;
          l_run += e;
        }
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        u32x4 vs[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          vs[j] = *reinterpret_cast<const u32x4*>(stage + St::kSteps + 128 * (kG + gr) + 32 * h + 16 * j);
        if (edge) {  // a token that is not seen may have any step: it counts as 0
#pragma unroll
          for (int j = 0; j < 16; j += 2)
            vs[j / 8][j / 2 % 4] &= ((uint32_t)__builtin_amdgcn_sbfe((int)seen, j, 1) & 0xFFFFu) |
                                    ((uint32_t)__builtin_amdgcn_sbfe((int)seen, j + 1, 1) & 0xFFFF0000u);
        }
        // P s in bf16 terms, tokens 16 h + 0..7 and 8..15.
        bf16x8 pf[2][kPT];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float step = step_of(vs[j / 8][j / 2 % 4], j & 1);
          __bf16 t[kPT];
          terms(p[j] * step, t);
#pragma unroll
          for (int i = 0; i < kPT; ++i) pf[j / 8][i][j % 8] = t[i];
        }
#pragma unroll
        for (int bl = 4 * gr; bl < 4 * gr + 4; ++bl) {
          const int t = 16 * h + r16;
          const int at = St::kCodes + t * St::kRow + 16 * ((bl >> 1) ^ St::value_swz(t)) + 8 * (bl & 1);
          const i32x2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(stage + at));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bf16x8 vf = numbers((uint32_t)w[u]);
#pragma unroll
            for (int i = 0; i < kPT; ++i) o[bl] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[u][i], o[bl], 0, 0, 0);
          }
        }
      }
      now ^= 1;
      number = next_number;
      next_number = after;
    }

    // Join the waves: unnormalised sums, maxima and weights through LDS.
    l_run = sum_halves(sum_rows16(l_run));
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds) + (size_t)wave * kTileRows * (D + 4);
#pragma unroll
    for (int bl = 0; bl < kB; ++bl) *reinterpret_cast<floatx4*>(sums + r16 * (D + 4) + 16 * bl + 4 * h) = o[bl];
    if (h == 0) {
      sums[r16 * (D + 4) + D] = m_run;
      sums[r16 * (D + 4) + D + 1] = l_run;
    }
    __syncthreads();
    for (int e = (int)threadIdx.x; e < kTileRows * D; e += 64 * kWaves) {
      const int tr = e / D, d = e % D;
      const int xe = x0 + tr;
      if (xe >= pairs) break;
      const float* all = reinterpret_cast<const float*>(lds) + tr * (D + 4);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, all[w * kTileRows * (D + 4) + D]);
      float sum = 0.0f, weight = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float* a = all + w * kTileRows * (D + 4);
        const float f = a[D] == top ? 1.0f : __builtin_amdgcn_exp2f((a[D] - top) * g.scale_log2);
        sum = __builtin_fmaf(a[d], f, sum);
        weight = __builtin_fmaf(a[D + 1], f, weight);
      }
      const int in_seq = g.over_group(xe), er = sq.first + in_seq, eh = head * g.group + xe - in_seq * g.group;
      if (tl.splits > 1) {
        const size_t at = ((size_t)split * g.rows + er) * g.q_heads + eh;
        g.part[at * D + d] = sum;
        if (d == 0) reinterpret_cast<float2*>(ends(g))[at] = make_float2(top, weight);
      } else {
        const float v = weight == 0.0f ? 0.0f : sum / weight;
        const size_t at = (size_t)er * g.out_stride + (size_t)eh * D + d;
        if constexpr (kF32)
          static_cast<float*>(g.out)[at] = v;
        else
          static_cast<__bf16*>(g.out)[at] = (__bf16)v;
      }
    }
    __syncthreads();
  }
}

// One workgroup a row and query head joins the splits' sums.  Its threads are D / 4 columns of
// four channels times kParts: part i adds splits i, i + kParts, ..., the parts are added in
// order.  Bound by latency: maxima and weights come in one load a lane, sums four at a time.
template <bool kF32, int D>
__global__ __launch_bounds__(256) void kv4_join_kernel(const Kv4Kernel g) {
  constexpr int kColumns = D / 4, kParts = 256 / kColumns;
  __shared__ floatx4 parts[kParts][kColumns];
  __shared__ float factors[kMaxSplits];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int column = tid % kColumns, part = tid / kColumns;
  const long long pairs = (long long)g.rows * g.q_heads;
  for (long long x = blockIdx.x; x < pairs; x += gridDim.x) {
    const int row = (int)(x / g.q_heads), q_head = (int)(x - (long long)row * g.q_heads);
    const int seq = find_sequence(g.starts, g.c.sequences, row);
    if (seq < 0) continue;
    const Sequence sq(g, seq);
    const int splits = Tile(g, sq, ((row - sq.first) * g.group + q_head % g.group) / kTileRows).splits;
    if (splits == 1) continue;
    float top = -INFINITY, weight = 0.0f;
    if (lane < splits) {
      const float2 e = reinterpret_cast<const float2*>(ends(g))[(size_t)lane * pairs + x];
      top = e.x;
      weight = e.y;
    }
    const float mine = top;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float f = mine == top ? 1.0f : __builtin_amdgcn_exp2f((mine - top) * g.scale_log2);
    weight = lane < splits ? weight * f : 0.0f;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) weight += __shfl_xor(weight, d);
    if (tid < splits) factors[tid] = f;
    __syncthreads();
    floatx4 sum = {};
    const floatx4* at = reinterpret_cast<const floatx4*>(g.part + (size_t)x * D) + column;
    const size_t slab = (size_t)pairs * kColumns;
#pragma unroll 4
    for (int s = part; s < splits; s += kParts) {
      const floatx4 v = at[s * slab];
      const float fs = factors[s];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(v[i], fs, sum[i]);
    }
    parts[part][column] = sum;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int i = 1; i < kParts; ++i) sum += parts[i][column];
      const size_t to = (size_t)row * g.out_stride + (size_t)q_head * D + 4 * column;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = weight == 0.0f ? 0.0f : sum[i] / weight;
        if constexpr (kF32)
          static_cast<float*>(g.out)[to + i] = v;
        else
          static_cast<__bf16*>(g.out)[to + i] = (__bf16)v;
      }
    }
    __syncthreads();
  }
}

// The grid: tiles of 16 pairs that the longest sequence has (a workgroup takes several where it
// would be too large), and splits for the pages of the longest.  A split has 4 to 32 pages (one to
// eight a wave), fewer where that is what fills the chip; a shorter sequence has fewer splits, so
// that workgroups are of one size whatever the lengths.
struct Plan {
  int tiles, splits, shift;
};
Plan plan(const Kv4AttentionArgs& a, int head_dim) {
  Plan p;
  const uint64_t columns = (uint64_t)a.c.sequences * a.c.kv_heads;  // at most kKv4MaxColumns
  const uint64_t t = ((uint64_t)a.max_rows * (uint64_t)a.group + kTileRows - 1) / kTileRows;
  p.tiles = (int)std::min<uint64_t>(t, kKv4MaxColumns / columns);
  uint64_t length = a.max_length;
  if (a.window) length = std::min<uint64_t>(length, (uint64_t)a.window + 2 * kKv4Page);
  const uint64_t pages = (length + kKv4Page - 1) / kKv4Page, base = columns * (uint64_t)p.tiles;
  p.shift = 2;
  while (p.shift < 5 && base * (pages >> p.shift) > 1024) ++p.shift;
  while (((pages + (1ull << p.shift) - 1) >> p.shift) > (uint64_t)kMaxSplits) ++p.shift;
  p.splits = (int)((pages + (1ull << p.shift) - 1) >> p.shift);
  if (base >= 4096 || (uint64_t)p.splits * a.rows * (uint64_t)a.q_heads * (uint64_t)(head_dim + 2) * 4 > kMostPartialBytes)
    p.splits = 1;
  return p;
}

template <bool kF32, int D>
hipError_t launch(const Kv4Kernel& g, hipStream_t stream) {
  const uint64_t grid = (uint64_t)g.c.sequences * g.c.kv_heads * (uint64_t)g.tiles * (uint64_t)g.splits;
  hipLaunchKernelGGL((kv4_attention_kernel<kF32, D>), dim3((unsigned)grid), dim3(64 * kWaves), 0, stream, g);
  if (g.splits > 1) {
    const uint64_t pairs = (uint64_t)g.rows * (uint64_t)g.q_heads;
    hipLaunchKernelGGL((kv4_join_kernel<kF32, D>), dim3((unsigned)std::min<uint64_t>(pairs, 1u << 20)), dim3(256),
                       0, stream, g);
  }
  return hipGetLastError();
}

}  // namespace

size_t kv4_attention_partial_bytes(const Kv4AttentionArgs& a, int head_dim) {
  const Plan p = plan(a, head_dim);
  return p.splits > 1 ? (size_t)p.splits * a.rows * a.q_heads * (head_dim + 2) * sizeof(float) : 0;
}

hipError_t launch_kv4_attention(const Kv4AttentionArgs& a, int head_dim, bool bf16, hipStream_t stream) {
  Kv4Kernel g{};
  g.c = a.c;
  g.q = a.q;
  g.out = a.out;
  g.starts = a.row_starts;
  g.part = a.part;
  g.rows = (int)a.rows;
  g.q_stride = (int)a.q_stride;
  g.out_stride = (int)a.out_stride;
  g.q_heads = a.q_heads;
  g.group = a.group;
  g.window = a.window > 0x7fffffffu ? 0 : (int)a.window;  // longer than any sequence
  g.scale_log2 = a.scale * 1.4426950408889634f;
  uint32_t l = 0;
  while ((1u << l) < (uint32_t)a.group) ++l;
  g.group_shift = 31 + l;
  g.group_magic = (1ull << g.group_shift) / (uint64_t)a.group + 1;
  const Plan p = plan(a, head_dim);
  g.tiles = p.tiles;
  g.splits = p.splits;
  g.split_shift = p.shift;
  g.ends = (size_t)p.splits * a.rows * (size_t)a.q_heads * (size_t)head_dim;
  switch (head_dim) {
    case 64: return bf16 ? launch<false, 64>(g, stream) : launch<true, 64>(g, stream);
    case 128: return bf16 ? launch<false, 128>(g, stream) : launch<true, 128>(g, stream);
    case 256: return bf16 ? launch<false, 256>(g, stream) : launch<true, 256>(g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace prom
