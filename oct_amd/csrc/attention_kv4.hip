// Attention over the 4-bit paged cache (kv4_cache.hip):
// o[r, h] = sum_t softmax_t(scale q[r, h] . k[t]) v[t], k[t] = s code, v[t] = s code
// with a step s for 64 channels of a token's head.
//
// Rows are (row, query head of the group) pairs, so that the heads that share a key head, and the
// rows of a prompt, read the cache once.  Two kernels.
//
// Few rows (decoding): a tile is 16 pairs, a wave takes a page (64 tokens) at a time, which it moves to
// its own part of LDS a page ahead (buffer_load ... lds, 16 bytes a lane; no wave waits for another).
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16.  E2M1 codes are exact in bf16 (one instruction turns two
//   codes into two numbers), so K goes into the products as codes, one accumulator a group of 64
//   channels, and the groups' steps are applied to the scores in fp32.  A lane owns one row and 16 of the
//   page's scores: tile c, register i of lane (h, row) is token 16 h + 4 c + i, so a lane's tokens are
//   neighbours and their steps four 16-byte loads.
//   Softmax in base 2 with a running maximum that follows only when it grew by more than 2^8.
//   O^T = V^T P^T.  V's step goes to the probability; P s is split into bf16 terms that carry it to 16
//   bits (24 for fp32 rows), the codes again are exact.  The V^T operand (16 channels, tokens in k) comes
//   from ds_read_b64_tr_b4, which hands a lane the 16 tokens of its channel; S^T's register order is
//   already P^T's operand order.  fp32 queries are three bf16 terms (exact).
// No rounding but P's and fp32's is made.  Pages of a sequence are dealt to the waves of a workgroup and
// to splits of the grid; the waves join through LDS, splits through fp32 partial sums and a second
// kernel, in a fixed order.  Bound by reading the cache, D + D / 16 bytes a token and key head: 64 rows over
// 64 sequences of up to 8192 tokens, 8 key heads of 128, groups of 4, bf16: 70 us, 4.6 TB/s, and 6 for the
// join; one row over 131072 tokens: 29 us, 4.9 TB/s, and 5.  A short sequence is bound by latency: 777
// tokens of one key head of 256, fp32, 9.5 us (a launch that does nothing 1.4, the way to the first page
// 2.5, a page 4, joining 1) and 4.
//
// Prompts: see kv4_prompt_kernel.
#include <algorithm>
#include <type_traits>

#include "lds_dma.h"
#include "reactor_internal.h"

namespace prom {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

constexpr float kLazyLog2 = 8.0f;
constexpr int kTileRows = 16;
constexpr int kWaves = 4;
// Sequences of up to kFewPairs pairs (rows times query heads of a group) stay on the kernel for few
// rows, whatever the call: a prompt tile has 128 or 256.  The prompts' kernel costs 40 to 85 us before
// it does much and then takes half the time for a page of 16 pairs, so it is taken from so many of
// them on (us with it / without, two prompts over up to 4096 tokens, 4 key heads, groups of 4; 256 and 118
// rows, 24064 pages of 16 pairs: bf16 64 channels 43 / 29, 128 56 / 49, 256 103 / 118, fp32 50 / 34,
// 65 / 62; 512 and 236 rows, 47872 pages: 48 / 50, 65 / 90, 147 / 222, 59 / 58, 94 / 114).  fp32 rows of
// 256 channels do not fit its registers (409 / 310).
constexpr uint64_t kFewPairs = 64;
constexpr uint64_t prompt_work(int head_dim) { return head_dim == 256 ? 24000 : 40000; }
constexpr int kMaxSplits = 64;  // a lane each when they are joined
constexpr int kPromptGroups = 256;  // workgroups that prompts are dealt to: one a CU
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
  int few_pairs;        // pairs (rows times group) up to which a sequence is not a prompt
  int join_heads;       // query heads that are joined at a time
  uint64_t* units;      // prompts: page units before each sequence, [sequences + 1]; null: no prompts
  float* prompt_part;   // sums [2 workgroups][rows of a tile][D], then (maximum, weight) of each
  size_t prompt_ends;   // where these begin
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

// A sequence's rows (those of the call's) and the first one's position, counted back from its length
// and the end of its rows, wherever that lies.
struct Sequence {
  int first, n, from;
  __device__ __forceinline__ Sequence(const Kv4Kernel& g, int seq) {
    Constant* starts = (Constant*)g.starts;
    const int end = starts[seq + 1];
    first = min(max(starts[seq], 0), g.rows);
    n = min(max(end, 0), g.rows) - first;
    from = max(((Constant*)g.c.lengths)[seq], 0) - (max(end, first) - first);
  }
};

// The tokens that a row sees, or is spoilt by: t with t - first < count (as unsigned numbers).
// On the page that stands for all behind the table (`past`) a row sees every token or none: one
// that lies there sees its own at least, which is bad.
struct Sees {
  uint32_t first, count;
  __device__ __forceinline__ Sees(const Kv4Kernel& g, int pos, bool past) {
    const int low = g.window && pos >= g.window ? pos - g.window + 1 : 0;
    first = past ? 0u : (uint32_t)low;
    count = past ? (pos / kKv4Page >= g.c.table_stride ? 0xFFFFFFFFu : 0u) : pos < low ? 0u : (uint32_t)(pos - low) + 1u;
  }
  __device__ __forceinline__ bool operator()(int t) const { return (uint32_t)t - first < count; }
};

// The positions of a tile's first and last row, the pages that they see between them, and into
// how many splits these are dealt.  Past the table every token is bad: the page behind its last
// stands for all of them.
struct Tile {
  int pos0, pos1, page0, last, splits;
  __device__ __forceinline__ Tile(const Kv4Kernel& g, const Sequence& s, int tile, int tile_rows = kTileRows) {
    const int x0 = tile * tile_rows;
    pos0 = s.from + g.over_group(x0);
    pos1 = s.from + g.over_group(min(x0 + tile_rows, s.n * g.group) - 1);
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
      lds_from_buffer(m0, off, d);
    }
  }
};

// Key heads fastest, then sequences, tiles, splits.  Workgroups go to the XCDs, and there to groups
// of CUs, in turn; the sequence moves on by one with each tile and split, so that the same CUs do
// not get every workgroup of a long sequence, or the splits that a short one does not have.
__device__ __forceinline__ void coordinates(const Kv4Kernel& g, int* head, int* seq, int* tile, int* split) {
  uint32_t b = blockIdx.x;
  *head = (int)(b % (uint32_t)g.c.kv_heads);
  b /= (uint32_t)g.c.kv_heads;
  const uint32_t i = b % (uint32_t)g.c.sequences;
  b /= (uint32_t)g.c.sequences;
  *tile = (int)(b % (uint32_t)g.tiles);
  *split = (int)(b / (uint32_t)g.tiles);
  *seq = (int)((i + (uint32_t)*tile + (uint32_t)*split) % (uint32_t)g.c.sequences);
}

// A prompt's work in units: a page of a tile (of Prompt::kRows pairs) of a key head.  All tiles of
// a sequence count the pages from its first tile's first to its last tile's last.
struct PromptSpan {
  int page0, pages, tiles;
  __device__ __forceinline__ PromptSpan(const Kv4Kernel& g, const Sequence& s, int tile_rows) {
    const int pairs = s.n * g.group;
    tiles = s.n > 0 && pairs > g.few_pairs ? (pairs + tile_rows - 1) / tile_rows : 0;
    page0 = pages = 0;
    if (tiles > 0) {
      page0 = Tile(g, s, 0, tile_rows).page0;
      pages = max(1, Tile(g, s, tiles - 1, tile_rows).last - page0);
    }
  }
};

// units[i] = units before sequence i: one workgroup of 256 threads, as many sequences at a time.
// waves: LDS of four numbers.
template <int kRows>
__device__ void count_prompt_units(const Kv4Kernel& g, uint64_t* waves) {
  const int tid = (int)threadIdx.x, lane = tid & 63;
  uint64_t before = 0;
  for (int from = 0; from < g.c.sequences; from += 256) {
    const int seq = from + tid;
    uint64_t own = 0;
    if (seq < g.c.sequences) {
      const PromptSpan span(g, Sequence(g, seq), kRows);
      own = (uint64_t)span.tiles * (uint64_t)span.pages * (uint64_t)g.c.kv_heads;
    }
    uint64_t sum = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 63) waves[tid >> 6] = sum;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < tid >> 6) sum += waves[w];
      all += waves[w];
    }
    if (seq < g.c.sequences) g.units[seq] = before + sum - own;
    before += all;
    __syncthreads();
  }
  if (tid == 0) g.units[g.c.sequences] = before;
}

// Waves of a prompt's workgroup, 32 pairs each: one or two a SIMD, by registers.
template <bool kF32, int D>
constexpr int kPromptWaves = D == 256 || (kF32 && D == 128) ? 4 : 8;

// The few rows' tiles; with prompts in the call, the last workgroup counts their units instead.
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
  if (g.units != nullptr && blockIdx.x == gridDim.x - 1) {
    static_assert(kWaves == 4, "units");
    count_prompt_units<32 * kPromptWaves<kF32, D>>(g, reinterpret_cast<uint64_t*>(lds));
    return;
  }
  int head, seq, tile0, split;
  coordinates(g, &head, &seq, &tile0, &split);
  const Sequence sq(g, seq);
  if (sq.n <= 0 || sq.n * g.group > g.few_pairs) return;
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
    const int pos = mine ? sq.from + row : tl.pos1;  // its position
    const int page0 = tl.page0, last = tl.last;

    // Q^T operand: lane (h, row), step s: channels 32 s + 8 h .. + 7.  Loaded here, used when the first
    // page is on its way.
    u32x4 q_raw[kSteps][kF32 ? 2 : 1];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const size_t at = (size_t)(sq.first + row) * g.q_stride + (size_t)q_head * D + 32 * s + 8 * h;
      if constexpr (kF32)
        __builtin_memcpy(q_raw[s], static_cast<const float*>(g.q) + at, 32);
      else
        __builtin_memcpy(q_raw[s], static_cast<const uint16_t*>(g.q) + at, 16);
    }
    __builtin_amdgcn_sched_barrier(0);

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
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 q[kSteps][kQT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          __bf16 t[kQT];
          terms(mine ? __uint_as_float(q_raw[s][j / 4][j % 4]) : 0.0f, t);
#pragma unroll
          for (int i = 0; i < kQT; ++i) q[s][i][j] = t[i];
        }
      } else {
        q[s][0] = __builtin_bit_cast(bf16x8, mine ? q_raw[s][0] : u32x4{0u, 0u, 0u, 0u});
      }
    }
    floatx4 o[kB] = {};
    float m_run = -INFINITY, m_log2 = 0.0f, l_run = 0.0f;
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
        const Sees row_sees(g, pos, past);
        const float poison = bad ? NAN : 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool sees = row_sees(t0 + 16 * h + 4 * c + i);
            s[c][i] = sees ? s[c][i] + poison : -INFINITY;
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
    // Four channels of a row a thread.
    static_assert(64 * kWaves * kG * 4 == kTileRows * D, "the tile's sums");
#pragma unroll
    for (int i = 0; i < kG; ++i) {
      const int e = (int)threadIdx.x + 64 * kWaves * i, tr = e / (D / 4), d = e % (D / 4) * 4;
      const int xe = x0 + tr;
      const float* all = reinterpret_cast<const float*>(lds) + tr * (D + 4);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, all[w * kTileRows * (D + 4) + D]);
      floatx4 sum = {};
      float weight = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float* a = all + w * kTileRows * (D + 4);
        const float f = a[D] == top ? 1.0f : __builtin_amdgcn_exp2f((a[D] - top) * g.scale_log2);
        const floatx4 v = *reinterpret_cast<const floatx4*>(a + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(v[j], f, sum[j]);
        weight = __builtin_fmaf(a[D + 1], f, weight);
      }
      if (xe >= pairs) continue;
      const int in_seq = g.over_group(xe), er = sq.first + in_seq, eh = head * g.group + xe - in_seq * g.group;
      if (tl.splits > 1) {
        const size_t at = ((size_t)split * g.rows + er) * g.q_heads + eh;
        *reinterpret_cast<floatx4*>(g.part + at * D + d) = sum;
        if (d == 0) reinterpret_cast<float2*>(ends(g))[at] = make_float2(top, weight);
      } else {
        const size_t at = (size_t)er * g.out_stride + (size_t)eh * D + d;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = weight == 0.0f ? 0.0f : sum[j] / weight;
        if constexpr (kF32) {
          __builtin_memcpy(static_cast<float*>(g.out) + at, v, 16);
        } else {
          const __bf16 b[4] = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
          __builtin_memcpy(static_cast<__bf16*>(g.out) + at, b, 8);
        }
      }
    }
    __syncthreads();
  }
}

// Many rows (prompts).  A workgroup takes 32 pairs a wave; a page's keys and values are turned
// into bf16 (exactly, steps applied) once for all of them and kept in LDS, and a wave computes
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_bf16, the V^T operand by transpose reads.
// The next page's codes are loaded into registers before a page is worked on and turned into the
// other half of LDS after it.  Of eight waves, the second of each SIMD runs half a page behind the first:
// one's products are beside the other's softmax.  P goes into the products as two bf16 terms (fp32 rows
// and their queries: three), as in the kernel for few rows, so that a call's precision does not
// depend on which of the two takes its sequences.  One term, 8 bits, added as much error as the results' own
// rounding (2.3e-3 of the values instead of 1.7e-3), and took 308 us instead of the 380 below.
// Bound by the matrix and vector units together, which two waves of a SIMD share less well than they
// could: four prompts of 1024 rows over up to 8000 tokens, 8 key heads of 128, groups of 4, bf16: 380 us for the
// call, 0.63 PFLOP/s of the definition's operations and half as many again for the second term (170 us at the rate of
// a large product).  A call of 350 us with one term, a part at a time: 65 without any of the four, 45 more with
// the loads, and beside these 35 with turning the codes, 78 with softmax, 153 with the products.
template <bool kF32, int D>
struct Prompt {
  static constexpr int kWaves = kPromptWaves<kF32, D>;
  static constexpr int kThreads = 64 * kWaves, kRows = 32 * kWaves;
  static constexpr int kUnits = 4 * D;                                // of 8 bytes (16 channels): keys, and values
  static constexpr int kEach = 2 * kUnits / kThreads > 0 ? 2 * kUnits / kThreads : 1;
  static constexpr int kTileBytes = kKv4Page * D * 2;                 // bf16 keys, or values
  static_assert(kEach * kThreads == 2 * kUnits && kUnits % 64 == 0, "units");

  // Position of 16-byte chunk c (8 channels) of token t: operand reads of 32 keys, and transpose
  // reads of 4 neighbouring tokens' 32 channels, then fall into different banks.
  __device__ static __forceinline__ int key_swz(int t) { return D == 64 ? t & 7 : t & 15; }
  __device__ static __forceinline__ int value_swz(int t) { return D == 64 ? 2 * t & 4 : 4 * (t & 3); }

  struct Codes {
    u32x2 w[kEach];
    uint32_t step[kEach];
  };
  __device__ static __forceinline__ void unit(int i, int tid, bool* keys, int* t, int* b) {
    const int u = tid + kThreads * i;
    *keys = u < kUnits;
    const int at = 8 * (u % kUnits);
    *t = at / (D / 2);
    *b = at % (D / 2);  // byte of the token's row
  }
  // Group of a unit: words of a key row lie four (D = 64: two) to a quarter, 32 channels apart.
  __device__ static __forceinline__ int group_of(bool keys, int b) {
    if (!keys) return b / 32;
    return D == 64 ? 0 : 2 * (b / 64) + b / 8 % 2;
  }
  // The thread's units of a keys' and a values' page.
  __device__ static __forceinline__ void load(Codes& c, const uint8_t* key_block, const uint8_t* value_block, int tid) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      bool keys;
      int t, b;
      unit(i, tid, &keys, &t, &b);
      const uint8_t* block = keys ? key_block : value_block;
      c.w[i] = *reinterpret_cast<const u32x2*>(block + (keys ? 0 : Stage<D>::kCodes) + t * (D / 2) + b);
      c.step[i] = *reinterpret_cast<const uint16_t*>(block + Stage<D>::kSteps + 128 * (group_of(keys, b) + (keys ? 0 : D / 64)) + 2 * t);
    }
  }
  // Codes to bf16 in LDS.  Values of an edge page, whose tokens some row does not see: those from token
  // zero_from of the page on, and those whose step is not finite, count as 0.  The one step that is larger than
  // kMostStep, 86 / 85 of it, would give infinities, and these NaN with a probability of 0.
  static constexpr int kMostStep = 0x7E2A0000;  // the largest that bf16 holds six of
  __device__ static __forceinline__ void store(const Codes& c, uint8_t* key_lds, uint8_t* value_lds, int tid, bool edge,
                                               int zero_from) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      bool keys;
      int t, b;
      unit(i, tid, &keys, &t, &b);
      uint32_t step = c.step[i] << 16;
      if (edge && !keys)
        step = t >= zero_from || (step & 0x7F800000u) == 0x7F800000u ? 0u : (uint32_t)min((int)step, kMostStep);
      const float s = __uint_as_float(step);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = c.w[i][j];
        const floatx2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
        const floatx2 v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
        const floatx2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
        const floatx2 v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        const bf16x8 x = {(__bf16)(v0.x * s), (__bf16)(v0.y * s), (__bf16)(v1.x * s), (__bf16)(v1.y * s),
                          (__bf16)(v2.x * s), (__bf16)(v2.y * s), (__bf16)(v3.x * s), (__bf16)(v3.y * s)};
        const int word = b / 4 + j;
        int chunk = word;
        if (keys) chunk = D == 64 ? 4 * (word & 1) + (word >> 1) : (word & ~15) + 4 * (word & 3) + (word >> 2 & 3);
        const int at = t * 2 * D + 16 * (chunk ^ (keys ? key_swz(t) : value_swz(t)));
        *reinterpret_cast<bf16x8*>((keys ? key_lds : value_lds) + at) = x;
      }
    }
  }
};

// A stretch of units within one tile and head: pages from..to of the sequence's span (0: its first).
struct PromptPiece {
  int seq, tile, head, from, to, pages;
  // The piece at unit u, cut at `end`.
  __device__ __forceinline__ PromptPiece(const Kv4Kernel& g, uint64_t u, uint64_t end, int tile_rows) {
    // The sequence: the last whose units begin at or before u (64 places a step); it has units,
    // since those without any begin where their successor does.
    const int lane = (int)threadIdx.x & 63;
    int lo = 0, span = g.c.sequences + 1;
    while (span > 1) {
      const int step = (span + 63) >> 6, at = lo + lane * step;
      const int c = __popcll(__ballot(at < lo + span && g.units[at] <= u));
      const int next = lo + (c - 1) * step;
      span = min(step, lo + span - next);
      lo = next;
    }
    seq = __builtin_amdgcn_readfirstlane(lo);
    const PromptSpan sp(g, Sequence(g, seq), tile_rows);
    pages = sp.pages;
    const uint64_t rel = u - g.units[seq];
    const uint64_t item = rel / (uint32_t)pages;
    from = __builtin_amdgcn_readfirstlane((int)(rel - item * (uint32_t)pages));
    const uint64_t left = end - u;
    to = left < (uint64_t)(pages - from) ? from + __builtin_amdgcn_readfirstlane((int)left) : pages;
    head = __builtin_amdgcn_readfirstlane((int)(item % (uint32_t)g.c.kv_heads));
    tile = __builtin_amdgcn_readfirstlane((int)(item / (uint32_t)g.c.kv_heads));
  }
};

// The first unit of workgroup w of n: shares that differ by one at most.
__device__ __forceinline__ uint64_t first_unit(uint64_t total, uint64_t w, uint64_t n) {
  return total / n * w + min(w, total % n);
}

// Workgroup w does units first_unit(w) to first_unit(w + 1), equal shares whatever tiles these cut through.
// A unit need not be a page that its tile sees (all tiles count the sequence's whole span), so that the shares of
// pages are even only where most of the span is seen: the busiest workgroup has 1.06 of the mean with four
// prompts of 1024 rows over 8000 tokens, but 1.94 to 1.99 with one of 2048 to 32768 rows and nothing before
// them (8 key heads, groups of 4; 4096 rows of 128 channels in bf16 320 us, 98 at the rate of a large product).  A
// piece that is not a whole tile leaves its sums in place 2 w + 1 where it begins the tile (it is then the
// workgroup's last), 2 w otherwise (its first), for join_prompts.
template <bool kF32, int D>
__global__ __launch_bounds__((Prompt<kF32, D>::kThreads), (Prompt<kF32, D>::kWaves / 4)) void kv4_prompt_kernel(const Kv4Kernel g) {
  using Pr = Prompt<kF32, D>;
  constexpr int kG = D / 64, kT = kF32 ? 3 : 1, kPT = kF32 ? 3 : 2;
  constexpr int kSteps = D / 16;  // MFMA steps of 16 channels
  constexpr int kB = D / 32;      // blocks of 32 output channels
  __shared__ __attribute__((aligned(1024))) uint8_t key_lds[2][Pr::kTileBytes], value_lds[2][Pr::kTileBytes];

  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31, hi = lane >> 5;
  const int behind = Pr::kWaves == 8 ? wave >> 2 : 0;  // half a page behind the other four waves
  const uint64_t total = g.units[g.c.sequences];
  uint64_t unit = first_unit(total, blockIdx.x, gridDim.x);
  const uint64_t unit_end = first_unit(total, blockIdx.x + 1ull, gridDim.x);
  while (unit < unit_end) {
    const PromptPiece piece(g, unit, unit_end, Pr::kRows);
    unit += (uint64_t)(piece.to - piece.from);
    const int head = piece.head, tile = piece.tile;
    const Sequence sq(g, piece.seq);
    const auto* table = (const Constant*)(g.c.table + (size_t)piece.seq * g.c.table_stride);
    const int pairs = sq.n * g.group;
    const Tile tl(g, sq, tile, Pr::kRows);
    const int span0 = PromptSpan(g, sq, Pr::kRows).page0;
    // This lane's row, and the first and last position of the wave's 32.
    const int x0 = tile * Pr::kRows + 32 * wave, x = x0 + lq;
    const bool mine = x < pairs;
    const int row = mine ? g.over_group(x) : 0;
    const int q_head = head * g.group + (mine ? x - row * g.group : 0);
    const int from = sq.from;
    const int wave0 = from + g.over_group(min(x0, pairs - 1)), wave1 = from + g.over_group(min(x0 + 32, pairs) - 1);
    const int pos = mine ? from + row : wave1;

    bf16x8 q[kSteps][kT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const size_t at = (size_t)(sq.first + row) * g.q_stride + (size_t)q_head * D + 16 * s + 8 * hi;
      if constexpr (kF32) {
        float v[8];
        __builtin_memcpy(v, static_cast<const float*>(g.q) + at, 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          __bf16 t[kT];
          terms(mine ? v[j] : 0.0f, t);
#pragma unroll
          for (int i = 0; i < kT; ++i) q[s][i][j] = t[i];
        }
      } else {
        u32x4 v;
        __builtin_memcpy(&v, static_cast<const uint16_t*>(g.q) + at, 16);
        if (!mine) v = u32x4{0u, 0u, 0u, 0u};
        q[s][0] = __builtin_bit_cast(bf16x8, v);
      }
    }

    floatx16 o[kB] = {};
    float m_run = -INFINITY, m_log2 = 0.0f, l_run = 0.0f;
    auto page_number = [&](int p) -> uint32_t {
      return p < tl.last && p < g.c.table_stride ? (uint32_t)table[p] : 0xFFFFFFFFu;
    };
    auto page_block = [&](uint32_t number) -> const uint8_t* {
      const uint32_t ok = number < g.c.pages ? number : 0u;
      return g.c.pool + ((size_t)ok * g.c.kv_heads + head) * kv4_block_bytes(D);
    };
    // Some row of the tile does not see all of the page.
    auto page_edge = [&](int p, uint32_t number) {
      return number >= g.c.pages || p * kKv4Page + (kKv4Page - 1) > tl.pos0 ||
             (g.window && p * kKv4Page <= tl.pos1 - g.window);
    };
    const int begin = max(tl.page0, span0 + piece.from), end = min(tl.last, span0 + piece.to);
    const int pages = end - begin;
    // Behind the last page the last one stands again, unused.
    auto number_of = [&](int n) { return page_number(begin + min(n, pages - 1)); };
    auto barrier = [] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    typename Pr::Codes codes;
    floatx16 s[2];
    bf16x8 p[4][kPT];
    // The matrix phase: O += V P of the page before and S = K Q of this one, in quads of four
    // operand reads and the instructions that use them; a quad is read while the one before it is
    // multiplied.  Operand e of the output: block e % kB of tokens 16 (e / kB) + 4 hi + 0..3 and 8
    // further; of the scores: step e / 2 of tokens 32 (e % 2) + lq.
    auto read_quad = [&](bf16x8 (&f)[4], int quad, const uint8_t* values, const uint8_t* keys) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * (quad % kB) + i;
        if (quad < kB) {
          const int t = 16 * (e / kB) + 4 * hi + ((lane & 15) >> 2);
          const int d = 32 * (e % kB) + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
          const uint8_t* at = values + t * 2 * D + 16 * ((d >> 3) ^ Pr::value_swz(t)) + 2 * (d & 7);
          const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
          const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * 2 * D));
          f[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
          const int t = 32 * (e % 2) + lq;
          f[i] = *reinterpret_cast<const bf16x8*>(keys + t * 2 * D + 16 * ((2 * (e / 2) + hi) ^ Pr::key_swz(t)));
        }
      }
    };
    auto use_quad = [&](const bf16x8 (&f)[4], int quad) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * (quad % kB) + i;
        if (quad < kB) {
#pragma unroll
          for (int j = 0; j < kPT; ++j) o[e % kB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i], p[e / kB][j], o[e % kB], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < kT; ++j) s[e % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i], q[e / 2][j], s[e % 2], 0, 0, 0);
        }
      }
    };
    auto multiply = [&](const uint8_t* values, const uint8_t* keys, auto scores) __attribute__((always_inline)) {
      constexpr int kQuads = decltype(scores)::value ? 2 * kB : kB;
      if constexpr (decltype(scores)::value) s[0] = s[1] = floatx16{};
      bf16x8 f[2][4];
      read_quad(f[0], 0, values, keys);
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        if (i + 1 < kQuads) read_quad(f[(i + 1) & 1], i + 1, values, keys);
        __builtin_amdgcn_sched_barrier(0);
        use_quad(f[i & 1], i);
      }
    };
    // Register r of block tb is token 32 tb + 8 (r / 4) + 4 hi + r % 4.
    auto weights = [&](int pg, uint32_t number) __attribute__((always_inline)) {
      const int t0 = pg * kKv4Page;
      const bool bad = number >= g.c.pages;
      const Sees row_sees(g, pos, pg >= g.c.table_stride);
      if (bad || t0 + (kKv4Page - 1) > wave0 || (g.window && t0 <= wave1 - g.window)) {
        const float poison = bad ? NAN : 0.0f;
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool sees = row_sees(t0 + 32 * tb + 8 * (r >> 2) + 4 * hi + (r & 3));
            s[tb][r] = sees ? s[tb][r] + poison : -INFINITY;
          }
      }
      float m = s[0][0];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, s[tb][r]);
      m = max_halves(m);
      if (__any((m - m_run) * g.scale_log2 > kLazyLog2)) {
        const float m_new = fmaxf(m, m_run);
        const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f((m_run - m_new) * g.scale_log2);
        m_run = m_new;
        m_log2 = m_new == -INFINITY ? 0.0f : m_new * g.scale_log2;
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < kB; ++i) o[i] *= alpha;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 2][8 * (c & 1) + j], g.scale_log2, -m_log2));
          l_run += e;
          __bf16 t[kPT];
          terms(e, t);
#pragma unroll
          for (int i = 0; i < kPT; ++i) p[c][i][j] = t[i];
        }
      // Values that are not finite are left out of an edge page: the rows that see them get NaN.
      if (!bad && page_edge(pg, number)) {
        const uint16_t* steps = reinterpret_cast<const uint16_t*>(page_block(number) + Stage<D>::kSteps + 2 * D) + lane;
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const uint64_t odd = __ballot((steps[64 * gr] & 0x7F80) == 0x7F80);
          if (odd != 0) {
            // The page's tokens that the row sees as bits.
            const uint32_t skip = row_sees.first > (uint32_t)t0 ? row_sees.first - t0 : 0u;
            const uint64_t upto = row_sees.first + row_sees.count - t0;  // tokens of the page before the end
            uint64_t sees = 0;
            if (row_sees.count != 0 && row_sees.first + row_sees.count > (uint32_t)t0 && skip < 64)
              sees = (upto >= 64 ? ~0ull : (1ull << upto) - 1) & (~0ull << skip);
            const float add = (odd & sees) != 0 ? NAN : 0.0f;
#pragma unroll
            for (int bl = 2 * gr; bl < 2 * gr + 2; ++bl) o[bl] += add;
          }
        }
      }
    };
    // A thread's units of keys' page n + 1 + behind and values' page n + behind, so that both are
    // whole before the first wave needs them and no half of LDS is written while it is read.
    auto convert = [&](int n, uint32_t value_number) __attribute__((always_inline)) {
      const int pg = begin + min(n + behind, pages - 1);
      Pr::store(codes, key_lds[(n + 1 + behind) & 1], value_lds[(n + behind) & 1], tid, page_edge(pg, value_number),
                value_number >= g.c.pages ? 0 : tl.pos1 - pg * kKv4Page + 1);
    };
    if (pages > 0) {
      uint32_t n0 = number_of(0), n1 = number_of(1), n2 = number_of(2);
      Pr::load(codes, page_block(n0), page_block(n0), tid);
      Pr::store(codes, key_lds[0], value_lds[1], tid, true, 0);  // keys; values of 0
      barrier();
      if (behind) {
        Pr::load(codes, page_block(n1), page_block(n0), tid);
        convert(-1, n0);
        barrier();
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < kPT; ++i) p[c][i] = bf16x8{};  // before the first page, with values of 0
      for (int n = 0; n < pages; ++n) {
        const uint32_t value_number = behind ? n1 : n0;
        Pr::load(codes, page_block(behind ? n2 : n1), page_block(value_number), tid);
        multiply(value_lds[(n + 1) & 1], key_lds[n & 1], std::true_type{});
        barrier();
        const uint32_t n3 = number_of(n + 3);  // here: the matrix phase's waits would wait for it
        weights(begin + n, n0);
        convert(n, value_number);
        barrier();
        n0 = n1;
        n1 = n2;
        n2 = n3;
      }
      multiply(value_lds[(pages + 1) & 1], nullptr, std::false_type{});
      barrier();
      if (Pr::kWaves == 8 && !behind) barrier();
    }

    l_run = sum_halves(l_run);
    if (mine) {
      if (piece.from > 0 || piece.to < piece.pages) {
        const size_t at = (2ull * blockIdx.x + (piece.from == 0)) * Pr::kRows + 32 * wave + lq;
#pragma unroll
        for (int bl = 0; bl < kB; ++bl)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            *reinterpret_cast<floatx4*>(g.prompt_part + at * D + 32 * bl + 8 * r + 4 * hi) =
                floatx4{o[bl][4 * r], o[bl][4 * r + 1], o[bl][4 * r + 2], o[bl][4 * r + 3]};
        if (hi == 0) reinterpret_cast<float2*>(g.prompt_part + g.prompt_ends)[at] = make_float2(m_run, l_run);
      } else {
        const float f = l_run == 0.0f ? 0.0f : 1.0f / l_run;
        const size_t at = (size_t)(sq.first + row) * g.out_stride + (size_t)q_head * D + 4 * hi;
#pragma unroll
        for (int bl = 0; bl < kB; ++bl)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (kF32) {
              const float v[4] = {o[bl][4 * r] * f, o[bl][4 * r + 1] * f, o[bl][4 * r + 2] * f, o[bl][4 * r + 3] * f};
              __builtin_memcpy(static_cast<float*>(g.out) + at + 32 * bl + 8 * r, v, 16);
            } else {
              const __bf16 v[4] = {(__bf16)(o[bl][4 * r] * f), (__bf16)(o[bl][4 * r + 1] * f),
                                   (__bf16)(o[bl][4 * r + 2] * f), (__bf16)(o[bl][4 * r + 3] * f)};
              __builtin_memcpy(static_cast<__bf16*>(g.out) + at + 32 * bl + 8 * r, v, 8);
            }
          }
      }
    }
  }
}

// Joins the pieces of a tile that workgroups of kv4_prompt_kernel cut it into, 16 rows a workgroup: workgroup
// `block` / (rows / 16)'s last piece if it begins a tile that the next workgroup goes on with, and the first
// pieces of those that follow up to the tile's end, in order.
template <bool kF32, int D>
__device__ void join_prompts(const Kv4Kernel& g, uint32_t block) {
  constexpr int kRows = Prompt<kF32, D>::kRows, kChannels = D / 16;
  const uint32_t part = block % (kRows / 16);
  const uint64_t total = g.units[g.c.sequences], n = kPromptGroups, w = block / (kRows / 16);
  const uint64_t begin = first_unit(total, w, n), end = first_unit(total, w + 1, n);
  if (begin == end) return;
  const PromptPiece last(g, end - 1, end, kRows);
  const uint64_t tile_begin = end - 1 - (uint64_t)last.from, tile_end = tile_begin + (uint64_t)last.pages;
  if (tile_begin < begin || tile_end == end) return;  // begun before, or whole
  uint64_t stop = w + 1;  // the workgroup behind the last that has a piece
  while (stop < n && first_unit(total, stop, n) < tile_end) ++stop;

  const Sequence sq(g, last.seq);
  const int r = 16 * (int)part + (int)threadIdx.x / 16, x = last.tile * kRows + r;
  if (x >= sq.n * g.group) return;
  const int row = g.over_group(x), q_head = last.head * g.group + x - row * g.group;
  const float2* all = reinterpret_cast<const float2*>(g.prompt_part + g.prompt_ends);
  auto place = [&](uint64_t i) { return (2 * i + (i == w)) * kRows + r; };
  float top = -INFINITY;
  for (uint64_t i = w; i < stop; ++i) top = fmaxf(top, all[place(i)].x);
  float sum[kChannels] = {}, weight = 0.0f;
  for (uint64_t i = w; i < stop; ++i) {
    const float2 e = all[place(i)];
    const float f = e.x == top ? 1.0f : __builtin_amdgcn_exp2f((e.x - top) * g.scale_log2);
    weight = __builtin_fmaf(e.y, f, weight);
    const float* from = g.prompt_part + place(i) * D + kChannels * (threadIdx.x % 16);
#pragma unroll
    for (int c = 0; c < kChannels; ++c) sum[c] = __builtin_fmaf(from[c], f, sum[c]);
  }
  const size_t to = (size_t)(sq.first + row) * g.out_stride + (size_t)q_head * D + kChannels * (threadIdx.x % 16);
#pragma unroll
  for (int c = 0; c < kChannels; ++c) {
    const float v = weight == 0.0f ? 0.0f : sum[c] / weight;
    if constexpr (kF32)
      static_cast<float*>(g.out)[to + c] = v;
    else
      static_cast<__bf16*>(g.out)[to + c] = (__bf16)v;
  }
}

// Joins the splits' sums: a workgroup a row, for every join_heads-th query head.  Its threads are D / 4 columns of
// four channels times kJoinParts: part i adds splits i, i + kJoinParts, ..., the parts are added in order.  Bound
// by latency: maxima and weights come in one load a lane, all sums at once beside them.  With no more splits than
// parts, a kernel of one sum a thread keeps twice the waves on a CU (64 rows of 32 heads of 128 in 4 splits 6.0 us,
// 8.2 with registers for 64; one row in 64 splits 4.9).
template <int D>
constexpr int kJoinParts = 256 / (D / 4);
// With prompts in the call, workgroups before those join their pieces: of one launch.
template <bool kF32, int D, int kEach>
__global__ __launch_bounds__(256) void kv4_join_kernel(const Kv4Kernel g) {
  uint32_t block = blockIdx.x;
  if constexpr (!kF32 || D != 256) {
    if (g.units != nullptr) {
      constexpr uint32_t kPromptBlocks = kPromptGroups * Prompt<kF32, D>::kRows / 16;
      if (block < kPromptBlocks) {
        join_prompts<kF32, D>(g, block);
        return;
      }
      block -= kPromptBlocks;
    }
  }
  constexpr int kColumns = D / 4, kParts = kJoinParts<D>;
  __shared__ floatx4 parts[kParts][kColumns];
  __shared__ float factors[kMaxSplits];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int column = tid % kColumns, part = tid / kColumns;
  const int row = (int)(block / (uint32_t)g.join_heads), head0 = (int)(block % (uint32_t)g.join_heads);
  const size_t pairs = (size_t)g.rows * g.q_heads;
  auto end_of = [&](int q_head) {  // of this lane's split, if there is one
    return lane < g.splits ? reinterpret_cast<const float2*>(ends(g))[lane * pairs + (size_t)row * g.q_heads + q_head]
                           : make_float2(-INFINITY, 0.0f);
  };
  float2 next = end_of(head0);
  const int seq = find_sequence(g.starts, g.c.sequences, row);
  if (seq < 0) return;
  const Sequence sq(g, seq);
  if (sq.n * g.group > g.few_pairs) return;
  for (int q_head = head0; q_head < g.q_heads; q_head += g.join_heads) {
    const size_t x = (size_t)row * g.q_heads + q_head;
    const float2 e = next;
    if (q_head + g.join_heads < g.q_heads) next = end_of(q_head + g.join_heads);
    // Splits that this row's tile does not have hold anything; they are left out.
    const int splits = Tile(g, sq, ((row - sq.first) * g.group + q_head % g.group) / kTileRows).splits;
    if (splits == 1) continue;
    // The sums, while the factors are worked out.
    floatx4 v[kEach];
    const floatx4* at = reinterpret_cast<const floatx4*>(g.part + (size_t)x * D) + column;
    const size_t slab = pairs * kColumns;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (part + kParts * i < splits) v[i] = at[(part + kParts * i) * slab];
    float top = lane < splits ? e.x : -INFINITY, weight = e.y;
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
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (part + kParts * i < splits) {
        const float fs = factors[part + kParts * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(v[i][j], fs, sum[j]);
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
  int tiles, splits, shift;  // of the sequences with few rows
  int few_pairs;             // up to so many pairs are few
  bool few;                  // there may be such sequences
  bool prompts;              // otherwise all rows go the way of few
  int prompt_rows;
  size_t prompt_ends;        // floats of the prompts' partial sums
  size_t part_bytes, prompt_bytes, unit_bytes;
};
Plan plan(const Kv4AttentionArgs& a, int head_dim, bool bf16) {
  Plan p{};
  const uint64_t columns = (uint64_t)a.c.sequences * a.c.kv_heads;  // at most kKv4MaxColumns
  const uint64_t most = (uint64_t)a.max_rows * (uint64_t)a.group;
  uint64_t length = a.max_length;
  if (a.window) length = std::min<uint64_t>(length, (uint64_t)a.window + a.max_rows + 2 * kKv4Page);
  const uint64_t small_tiles = ((uint64_t)a.rows * (uint64_t)a.group + kTileRows - 1) / kTileRows;
  const uint64_t work = small_tiles * (uint64_t)a.c.kv_heads * ((length + kKv4Page - 1) / kKv4Page);
  if (most > kFewPairs && work > prompt_work(head_dim) && (bf16 || head_dim != 256)) {
    p.prompt_rows = 32 * (head_dim == 256 || (!bf16 && head_dim == 128) ? 4 : 8);
    p.prompts = true;
    p.prompt_ends = 2ull * kPromptGroups * p.prompt_rows * (size_t)head_dim;
    p.prompt_bytes = (p.prompt_ends + 4ull * kPromptGroups * p.prompt_rows) * sizeof(float);
    p.unit_bytes = ((size_t)a.c.sequences + 1) * sizeof(uint64_t);
  }
  // A call of one sequence is either; otherwise sequences of few rows go their own way beside prompts.
  p.few = !p.prompts || a.c.sequences > 1;
  p.few_pairs = !p.prompts ? 0x7fffffff : p.few ? (int)kFewPairs : 0;
  if (!p.few) return p;
  p.tiles = (int)std::min<uint64_t>((std::min<uint64_t>(most, p.few_pairs) + kTileRows - 1) / kTileRows, kKv4MaxColumns / columns);
  const uint64_t pages = (length + kKv4Page - 1) / kKv4Page, base = columns * (uint64_t)p.tiles;
  p.shift = 2;
  while (p.shift < 5 && base * (pages >> p.shift) > 1024) ++p.shift;
  while (((pages + (1ull << p.shift) - 1) >> p.shift) > (uint64_t)kMaxSplits) ++p.shift;
  p.splits = (int)((pages + (1ull << p.shift) - 1) >> p.shift);
  p.part_bytes = (size_t)p.splits * a.rows * (size_t)a.q_heads * (size_t)(head_dim + 2) * sizeof(float);
  // With very many workgroups, or more than 1 GiB of partial sums (which count every row of the call), none is
  // split: a few long sequences among many short ones, or beside a long prompt, are then a few workgroups' work
  // (bf16, 8 key heads of 128, groups of 4: 1024 rows 42 us, eight rows over 131072 tokens 261, both in a call 869;
  // 512 rows over 1000 tokens 117, with one of them over 131072 908).
  if (base >= 4096 || p.part_bytes > kMostPartialBytes) p.splits = 1;
  if (p.splits == 1) p.part_bytes = 0;
  return p;
}

template <bool kF32, int D>
hipError_t launch(Kv4Kernel g, const Plan& p, hipStream_t stream) {
  const unsigned tiles = p.few ? (unsigned)g.c.sequences * (unsigned)g.c.kv_heads * (unsigned)p.tiles * (unsigned)p.splits : 0u;
  hipLaunchKernelGGL((kv4_attention_kernel<kF32, D>), dim3(tiles + (p.prompts ? 1u : 0u)), dim3(64 * kWaves), 0, stream, g);
  unsigned joins = 0;
  if constexpr (!kF32 || D != 256) {
    if (p.prompts) {
      hipLaunchKernelGGL((kv4_prompt_kernel<kF32, D>), dim3(kPromptGroups), dim3((Prompt<kF32, D>::kThreads)), 0, stream, g);
      joins = kPromptGroups * Prompt<kF32, D>::kRows / 16;
    }
  }
  if (p.few && p.splits > 1) {
    g.join_heads = (int)std::min<unsigned>((unsigned)g.q_heads, std::max(1u, 4096u / (unsigned)g.rows));
    joins += (unsigned)g.rows * (unsigned)g.join_heads;
  }
  if (joins > 0) {
    if (p.splits <= kJoinParts<D>)
      hipLaunchKernelGGL((kv4_join_kernel<kF32, D, 1>), dim3(joins), dim3(256), 0, stream, g);
    else
      hipLaunchKernelGGL((kv4_join_kernel<kF32, D, kMaxSplits / kJoinParts<D>>), dim3(joins), dim3(256), 0, stream, g);
  }
  return hipGetLastError();
}

size_t round_up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

}  // namespace

size_t kv4_attention_partial_bytes(const Kv4AttentionArgs& a, int head_dim, bool bf16) {
  const Plan p = plan(a, head_dim, bf16);
  return round_up(p.part_bytes) + round_up(p.prompt_bytes) + p.unit_bytes;
}

hipError_t launch_kv4_attention(const Kv4AttentionArgs& a, int head_dim, bool bf16, hipStream_t stream) {
  Kv4Kernel g{};
  g.c = a.c;
  g.q = a.q;
  g.out = a.out;
  g.starts = a.row_starts;
  g.rows = (int)a.rows;
  g.q_stride = (int)a.q_stride;
  g.out_stride = (int)a.out_stride;
  g.q_heads = a.q_heads;
  g.group = a.group;
  g.window = a.window > 0x7fffffffu ? 0 : (int)a.window;  // longer than any sequence
  g.scale_log2 = a.scale * kLog2E;
  uint32_t l = 0;
  while ((1u << l) < (uint32_t)a.group) ++l;
  g.group_shift = 31 + l;
  g.group_magic = (1ull << g.group_shift) / (uint64_t)a.group + 1;
  const Plan p = plan(a, head_dim, bf16);
  g.tiles = p.tiles;
  g.splits = p.splits;
  g.split_shift = p.shift;
  g.few_pairs = p.few_pairs;
  g.part = a.part;
  g.ends = (size_t)p.splits * a.rows * (size_t)a.q_heads * (size_t)head_dim;
  g.prompt_part = reinterpret_cast<float*>(reinterpret_cast<char*>(a.part) + round_up(p.part_bytes));
  g.prompt_ends = p.prompt_ends;
  if (p.prompts) g.units = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(g.prompt_part) + round_up(p.prompt_bytes));
  switch (head_dim) {
    case 64: return bf16 ? launch<false, 64>(g, p, stream) : launch<true, 64>(g, p, stream);
    case 128: return bf16 ? launch<false, 128>(g, p, stream) : launch<true, 128>(g, p, stream);
    case 256: return bf16 ? launch<false, 256>(g, p, stream) : launch<true, 256>(g, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace prom
