// The product with 4-bit weights: c[i, j] = sum_k x[i, k] w[j, k], w as w4_tiles.h lays it out.
//
// Few rows: bound by reading w, and by latency where it is small.  A workgroup takes kNT tiles of 16 columns, its waves
// every kWaves-th tile of K each (memory is read in order by the workgroup), and adds their sums through LDS.  Where
// columns are few, K is cut into slices over workgroups too: each leaves its sums in memory and the last one to do so adds
// them, in their order.  bf16, 32768x2048 in groups of 128, one row: 7.1 us, 35 MB at 4.9 TB/s (a large copy runs at
// 5.1).  fp32, 15 rows, 2048x16384 in groups of 32: 12.6 us for 20 MB, most of it latency: the loads, the split into terms, two
// joins.
//
// Many rows: a workgroup's four waves take 16 kMT rows by 64 kNT columns.  x goes to LDS by DMA, in the order in which
// the matrix units take it (1 KiB a transfer, each lane its own 16 bytes of source), a tile of K ahead; each wave holds its
// columns' codes in registers and turns them into bf16 weights, code times step, between its matrix instructions (four
// vector instructions for two weights, used for kMT blocks of rows).  Bound by the SIMDs, whose matrix instructions and
// conversions take turns, and by the last round: bf16, 512 rows of 20480x3840 86 us, 936 TFLOP/s, of which the matrix
// instructions alone take 69; its 428 workgroups leave 84 CUs with one for two places, done after 51 of 85 us of K tiles.  A large
// bf16 product runs at 1256.
#include <algorithm>

#include "fp4_groups.h"
#include "lds_dma.h"
#include "reactor_internal.h"
#include "tickets.h"
#include "w4_product.h"

namespace prom {
namespace {

struct W4Args {
  W4View w;
  const void* x;
  void* out;
  float* part;  // slices' sums, [workgroup of a slice][slice][row][16 kNT]
  uint32_t x_stride, out_stride;
  int m, slices;
};

constexpr int kTickets = 1024, kMaxSlices = 8;
constexpr uint32_t kMaxTileStride = 1u << 22;  // byte offsets within a tile's rows fit 31 bits
__device__ uint32_t w4_tickets[kTickets];

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

// grid.x: column groups times blocks of sixteen rows; those of one group are neighbours on one XCD, so that its L2
// brings their weights once.  grid.y: slices.
template <typename X, int kSteps, int kNT, int kWaves, W4Edge kEdge>
__global__ __launch_bounds__(64 * kWaves) void w4_rows_kernel(const W4Args a) {
  typedef typename X::Element T;
  constexpr int kPart = 256 * kNT;
  __shared__ float sums[kWaves][kNT][4][64];
  __shared__ uint32_t ticket;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int blocks = (a.m + 15) >> 4;
  const int id = blocks > 1 ? xcd_pid((int)blockIdx.x, (int)gridDim.x) : (int)blockIdx.x;
  const int group = id / blocks, row0 = 16 * (id - group * blocks), rows = min(a.m - row0, 16);
  const u32x4* codes[kNT];
  const uint16_t* steps[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    const int tile = min(group * kNT + i, a.w.tiles_n - 1);
    codes[i] = w4_codes(a.w, 0, tile);
    steps[i] = w4_steps<kSteps>(a.w, 0, tile);
  }
  floatx4 acc[1][kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) acc[0][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  // Slice y of K: tiles begin .. end - 1 (at most 2^13 tiles).
  const int slice = (int)blockIdx.y;
  const int begin = a.w.tiles_k * slice / a.slices, end = a.w.tiles_k * (slice + 1) / a.slices;
  W4Tile<kSteps, kNT> first;
  first.fetch(codes, steps, min(begin + wave, end - 1));
  X x[1];
  x[0].p = static_cast<const T*>(a.x) + (size_t)(row0 + min(lane & 15, rows - 1)) * a.x_stride;
  w4_accumulate<kSteps, kNT, 1, kEdge>(codes, steps, first, x, begin + wave, end, kWaves, a.w.k, acc);
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][i][r][lane] = acc[0][i][r];
  __syncthreads();
  const int column0 = group * kNT * kW4TileN, count = rows * kNT * 16;
  T* out = static_cast<T*>(a.out) + (size_t)row0 * a.out_stride + column0;
  float* part = a.slices > 1 ? a.part + (size_t)id * a.slices * kPart : nullptr;
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    const int row = at / (16 * kNT), c = at % (16 * kNT), r = row & 3, l = 16 * (row >> 2) + (c & 15);
    float v = sums[0][c >> 4][r][l];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][c >> 4][r][l];
    if (part != nullptr)
      __hip_atomic_store(part + (size_t)slice * kPart + at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else if (column0 + c < a.w.n)
      put(out + (size_t)row * a.out_stride + c, v);
  }
  if (part == nullptr || !last_to_arrive(w4_tickets + id, (uint32_t)a.slices, &ticket)) return;
  for (int at = (int)threadIdx.x; at < count; at += 64 * kWaves) {
    const int row = at / (16 * kNT), c = at % (16 * kNT);
    float p[kMaxSlices];
#pragma unroll
    for (int s = 0; s < kMaxSlices; ++s)
      p[s] = s < a.slices ? __hip_atomic_load(part + (size_t)s * kPart + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f;
    float v = p[0];
#pragma unroll
    for (int s = 1; s < kMaxSlices; ++s) v += p[s];
    if (column0 + c < a.w.n) put(out + (size_t)row * a.out_stride + c, v);
  }
}

__device__ __forceinline__ void put8(float* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = v[j];
  }
}
__device__ __forceinline__ void put8(uint16_t* p, int left, const float (&v)[8]) {
  __bf16 w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = (__bf16)v[j];
  if (left >= 8) {
    __builtin_memcpy(p, w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = __builtin_bit_cast(uint16_t, w[j]);
  }
}

// ------------------------------------------------------------------ many rows
struct W4TileArgs {
  W4View w;
  const uint16_t* x;   // kTerms planes of bf16 rows, `plane` elements apart, rows of ld (16-byte aligned)
  void* out;
  size_t plane;
  uint32_t out_stride;
  int m, ld, k;        // k columns of x are valid, a multiple of 8
  int tiles_m, tiles_n;
};

template <int kN>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kN) : "memory");
}

// Eight weights of a column: codes times the group's step, exact in bf16 (a step has six significant bits, a code two).
__device__ __forceinline__ bf16x8 w4_weights(uint32_t codes, float step) {
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const floatx2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const floatx2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  const auto pair = [&](floatx2 v) {
    return __builtin_amdgcn_perm(__float_as_uint(v.y * step), __float_as_uint(v.x * step), 0x07060302u);
  };
  return __builtin_bit_cast(bf16x8, u32x4{pair(a), pair(b), pair(c), pair(d)});
}

template <int kSteps, int kNT, int kMT, int kTerms, typename T>
__global__ __launch_bounds__(256, 2) void w4_tile_kernel(const W4TileArgs a) {
  constexpr int kStage = kTerms * kMT * 4096, kPitch = 16 * kNT + 4;
  constexpr int kLds = 2 * kStage > 4 * 16 * kPitch * 4 ? 2 * kStage : 4 * 16 * kPitch * 4;
  static_assert(2 * kLds <= 163840, "two workgroups a CU");
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int pid = xcd_pid((int)blockIdx.x, a.tiles_m * a.tiles_n);
  const int tm = pid % a.tiles_m, tn = pid / a.tiles_m;
  const int row0 = tm * 16 * kMT, rows = min(a.m - row0, 16 * kMT);
  const int tile0 = (tn * 4 + wave) * kNT;  // this wave's first tile of columns
  const int tiles_k = a.w.tiles_k;

  // x: this wave brings step u = wave of each block of sixteen rows, 1 KiB in the order of the matrix units.
  const uint32_t x_off = (uint32_t)(lane & 15) * (uint32_t)a.ld * 2u + (uint32_t)(32 * wave + 8 * (lane >> 4)) * 2u;
  const uint32_t block = 16u * (uint32_t)a.ld * 2u;
  const uint32_t range = ((uint32_t)(rows - 1) * (uint32_t)a.ld + (uint32_t)a.k) * 2u;
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
  const auto bring = [&](int kt, uint32_t stage) __attribute__((always_inline)) {
    // columns from k on: past every range, which brings zeros
    const int column = kt * kW4TileK + 32 * wave + 8 * (lane >> 4);
    const uint32_t at = column < a.k ? x_off + (uint32_t)kt * (2 * kW4TileK) : 0x80000000u;
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
      const unsigned long long base = (unsigned long long)(a.x + t * a.plane + (size_t)row0 * a.ld);
      typedef int intx4 __attribute__((ext_vector_type(4)));
      intx4 d;
      d.x = __builtin_amdgcn_readfirstlane((int)(base & 0xffffffffu));
      d.y = __builtin_amdgcn_readfirstlane((int)(base >> 32));
      d.z = __builtin_amdgcn_readfirstlane((int)range);
      d.w = 0x00020000;
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + stage + (uint32_t)((t * kMT + m) * 4 + wave) * 1024u);
        const uint32_t off = at + (uint32_t)m * block;
        lds_from_buffer(to, off, d);
      }
    }
  };

  const u32x4* codes[kNT];
  const uint16_t* steps[kNT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) {
    const int tile = min(tile0 + i, a.w.tiles_n - 1);
    codes[i] = w4_codes(a.w, 0, tile);
    steps[i] = w4_steps<kSteps>(a.w, 0, tile);
  }
  floatx4 acc[kMT][kNT];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int i = 0; i < kNT; ++i) acc[m][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  // A tile of K is 4 kTerms steps; a step's operands are read and turned into bf16 during the step before, between
  // its matrix instructions.  Before the last step of a tile the next one's x has to be there; its weights come with it.
  W4Tile<kSteps, kNT> now, next;
  const auto settle = [&](W4Tile<kSteps, kNT>& w) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kNT; ++i) {  // here, where they have arrived: behind later loads they would wait for those
      asm volatile("" : "+v"(w.c[i]));
#pragma unroll
      for (int v = 0; v < (int)(sizeof(w.s[i].v) / 4); ++v) asm volatile("" : "+v"(w.s[i].v[v]));
    }
  };
  const auto read = [&](uint32_t from, int q, bf16x8 (&to)[kMT]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < kMT; ++m)
      to[m] = *reinterpret_cast<const bf16x8*>(lds + from + (((kTerms - 1 - q % kTerms) * kMT + m) * 4 + q / kTerms) * 1024 +
                                               lane * 16);
  };
  const auto turn = [&](const W4Tile<kSteps, kNT>& w, int u, bf16x8 (&to)[kNT]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kNT; ++i) to[i] = w4_weights(w.c[i][u], w.s[i][u * kSteps / 4]);
  };
  constexpr int kQ = 4 * kTerms;
  bf16x8 x[2][kMT], b[2][kNT];
  uint32_t stage = 0;
  now.fetch(codes, steps, 0);
  bring(0, 0);
  next.fetch(codes, steps, min(1, tiles_k - 1));
  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  settle(now);
  settle(next);
  if (tiles_k > 1) bring(1, (uint32_t)kStage);
  read(0, 0, x[0]);
  turn(now, 0, b[0]);
#pragma unroll 1
  for (int kt = 0; kt < tiles_k; ++kt) {
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const int u = q / kTerms;
      __builtin_amdgcn_sched_barrier(0);
      if (q == kQ - 1) {
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // x of the next tile is there for all waves, this tile's is read
        asm volatile("" ::: "memory");
        settle(next);
        now = next;
        if (kt + 2 < tiles_k) bring(kt + 2, stage);
        next.fetch(codes, steps, min(kt + 2, tiles_k - 1));
        asm volatile("" ::: "memory");  // the loads above stay above: the compiler would move them to their use
        stage ^= (uint32_t)kStage;
      }
      __builtin_amdgcn_sched_barrier(0);
      read(stage, (q + 1) % kQ, x[(q + 1) & 1]);
      if ((q + 1) % kTerms == 0) turn(now, (u + 1) % 4, b[(u + 1) & 1]);
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int i = 0; i < kNT; ++i)
          acc[m][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[q & 1][m], b[u & 1][i], acc[m][i], 0, 0, 0);
#pragma unroll
      for (int m = 0; m < kMT; ++m) {  // a read, then matrix instructions with vector ones between them
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if ((q + 1) % kTerms == 0) __builtin_amdgcn_sched_group_barrier(0x002, (16 + kMT - 1) / kMT, 0);
        }
      }
    }
  }
  // Sixteen rows of the wave's columns at a time go through its part of LDS, so that a lane stores eight values of a row.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  float* mine = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
#pragma unroll
  for (int m = 0; m < kMT; ++m) {
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[(4 * (lane >> 4) + r) * kPitch + 16 * i + (lane & 15)] = acc[m][i][r];
    asm volatile("" ::: "memory");  // a wave's own part: its LDS operations stay in order
#pragma unroll
    for (int j = 0; j < (32 * kNT + 63) / 64; ++j) {
      const int item = j * 64 + lane, r = item / (2 * kNT), c = item % (2 * kNT) * 8;
      const int row = 16 * m + r, column = tile0 * kW4TileN + c;
      if (item < 32 * kNT && row < rows && column < a.w.n) {
        float v[8];
        __builtin_memcpy(v, __builtin_assume_aligned(mine + r * kPitch + c, 16), 32);
        put8(static_cast<T*>(a.out) + (size_t)(row0 + row) * a.out_stride + column, a.w.n - column, v);
      }
    }
    asm volatile("" ::: "memory");
  }
}

// Rows as bf16 terms, aligned and zero-padded to ld columns: what the tiles' DMA takes.
template <typename X>
__global__ __launch_bounds__(256) void w4_terms_kernel(const void* __restrict__ x, uint32_t stride, uint16_t* __restrict__ to,
                                                       size_t plane, int m, int k, int ld) {
  typedef typename X::Element T;
  constexpr W4Edge kTermsEdge = sizeof(T) == 2 ? kEdgeOdd : kEdgeNone;
  const int c = (int)(blockIdx.x * 64 + (threadIdx.x & 63)) * 8;
  if (c >= ld) return;
  for (int r = (int)(blockIdx.y * 4 + (threadIdx.x >> 6)); r < m; r += (int)gridDim.y * 4) {
    X row;
    row.p = static_cast<const T*>(x) + (size_t)r * stride;
    typename X::Raw raw = c + 8 <= k ? row.template fetch<kTermsEdge>(c, k) : row.template fetch<kEdgeShort>(c, k);
    bf16x8 t[X::kTerms];
    X::terms(raw, t);
#pragma unroll
    for (int i = 0; i < X::kTerms; ++i)
      *reinterpret_cast<bf16x8*>(to + i * plane + (size_t)r * ld + c) = t[i];
  }
}

struct RowsPlan {
  int nt, waves, slices;
};

// A launch wants a workgroup on most of the 256 CUs (kMostCus of them will do), and as many columns a workgroup as that
// leaves: they share the rows' operands.  us, bf16: 12288x4096, one row, 64, 32 or 16 columns 7.3, 8.1, 9.2; 8192x2048
// 4.7, 4.2, 5.1; 4096x4096, 16 rows 7.9 to 8.8, 7.1 to 7.5, 6.9, 64 rows 8.7, 12, 21; 33 rows of 3008x1920 5.5, 7.2, 8.5.
// Where even 16 columns leave CUs idle and K is long it is cut: 2048x16384, one row 13.2 in one slice, 7.4 in four.  fp32
// rows take three times the matrix instructions and have to be split into terms, so that more columns share that and
// shorter K are cut: 15 rows of 2048x2048 7.4, 6.0 in four slices; 16 rows of 4096x4096 11.5 with 16 columns, 8.7 with 64 in
// four slices.  Eight waves a workgroup where each has a CU: 12288x4096 7.3, with four 8.1; four where some would wait for
// a second round: 20480x2048 8.1 with eight, 7.5; 16 fp32 rows of 17920x1024 12.1 and 9.1.
// Two or one where there are many, whose sums are joined and stored while others multiply: 64 rows of 16384x2048 16.7 with
// four waves, 14.1 with two, 16.0 with one; of 32768x2048 29, 30 and 24; fp32 rows the same, but 64 of 12288x4096 32.6 and 35.4.
RowsPlan plan_rows(uint32_t m, const W4View& w, bool bf16) {
  constexpr int kMostCus = 140;
  const int blocks = (int)((m + 15) / 16);
  const auto groups = [&](int nt) { return (w.tiles_n + nt - 1) / nt * blocks; };
  const bool cut = groups(1) < kMostCus || !bf16;
  RowsPlan p{1, 8, 1};
  if (groups(4) >= kMostCus || (!bf16 && groups(2) < kMostCus && w.tiles_k >= 32))
    p.nt = 4;
  else if (groups(2) >= kMostCus || !bf16 || (cut && w.tiles_k >= 64))
    p.nt = 2;
  if (p.nt == 4)
    p.waves = groups(4) >= 2000 ? 1 : groups(4) >= (bf16 ? 768 : 800) ? 2 : groups(4) > 256 ? 4 : 8;
  else if (p.nt == 2 && bf16)
    p.waves = 4;
  if (cut && groups(p.nt) < kMostCus && w.tiles_k >= (bf16 ? 64 : 16))
    while (p.slices < kMaxSlices && groups(p.nt) * p.slices <= 128 && w.tiles_k >= 8 * p.slices) p.slices *= 2;
  return p;
}

template <typename X, int kSteps, W4Edge kEdge>
hipError_t launch_rows(const RowsPlan& p, const W4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.w.tiles_n + p.nt - 1) / p.nt) * (unsigned)((a.m + 15) / 16), (unsigned)a.slices);
#define ROWS(NT, W)                                                                                                  \
  if (p.nt == NT && p.waves == W)                                                                                    \
    hipLaunchKernelGGL((w4_rows_kernel<X, kSteps, NT, W, kEdge>), grid, dim3(64 * W), 0, stream, a);
  if constexpr (X::kTerms == 1) {
    ROWS(1, 8) ROWS(2, 4)
  } else {
    ROWS(2, 8)
  }
  ROWS(4, 1) ROWS(4, 2) ROWS(4, 4) ROWS(4, 8)
#undef ROWS
  return hipGetLastError();
}

template <typename X, int kSteps>
hipError_t launch_rows(const RowsPlan& p, const W4Args& a, hipStream_t stream) {
  const W4Edge edge = w4_edge<typename X::Element>(a.x, a.x_stride, a.w.k);
  if (edge == kEdgeNone) return launch_rows<X, kSteps, kEdgeNone>(p, a, stream);
  if (edge == kEdgeShift) return launch_rows<X, kSteps, kEdgeShift>(p, a, stream);
  if constexpr (sizeof(typename X::Element) == 2)
    if (edge == kEdgeOdd) return launch_rows<X, kSteps, kEdgeOdd>(p, a, stream);
  hipLaunchKernelGGL((w4_rows_kernel<X, kSteps, 1, 8, kEdgeShort>),
                     dim3((unsigned)a.w.tiles_n * (unsigned)((a.m + 15) / 16)), dim3(512), 0, stream, a);
  return hipGetLastError();
}

// Microseconds of a tile of K for a workgroup alone on its CU and for two that share one, bf16 and fp32 (three terms),
// from products of 2048 to 4096 columns and rows that make one round, two and more.
struct TileCost {
  int nt, mt;
  double alone, pair;
};
constexpr TileCost kTiles[] = {{2, 4, 0.86, 1.25}, {4, 4, 1.35, 2.24}, {3, 8, 1.70, 2.84}};
constexpr TileCost kTilesF32[] = {{2, 2, 1.04, 1.67}, {4, 2, 1.66, 2.76}};

struct TilePlan {
  int nt, mt;
  double us;
};
template <size_t kN>
TilePlan plan_tiles(const TileCost (&costs)[kN], uint32_t m, const W4View& w) {
  TilePlan best{0, 0, 1e300};
  for (const TileCost& c : costs) {
    const uint64_t wgs = (uint64_t)((m + 16u * c.mt - 1) / (16u * c.mt)) * (unsigned)((w.tiles_n + 4 * c.nt - 1) / (4 * c.nt));
    const uint64_t rest = wgs % 512;
    const double us = 4.0 + w.tiles_k * ((double)(wgs / 512) * c.pair + (rest == 0 ? 0.0 : rest <= 256 ? c.alone : c.pair));
    if (us < best.us) best = TilePlan{c.nt, c.mt, us};
  }
  return best;
}
// `terms`: x has to be brought into terms first, in a launch of its own.
TilePlan plan_tiles(uint32_t m, const W4View& w, bool bf16, bool terms) {
  TilePlan p = bf16 ? plan_tiles(kTiles, m, w) : plan_tiles(kTilesF32, m, w);
  p.us += 4.5e-7 * m * w.n + (terms ? 3.0 : 0.0);  // storing the result
  return p;
}
// Whether the few rows' kernel, which reads the weights again for each sixteen rows, is the shorter way: a launch, its
// workgroups' ends and the products, from 180 to 400 rows of 2048 and 15008 by 128 to 8192 (bf16, 180 rows of 15008x128 7.8 us,
// on tiles 6.2; 400 of 2048x1024 8.7 and 9.6).  Both ways were timed from 66 rows on; up to 64 it is taken without asking, also where
// the estimates say otherwise (64 rows of 32768x2048: 27.9 us and 18.7; it takes 24).
bool rows_are_few(uint32_t m, const W4View& w, bool bf16, const TilePlan& tiles) {
  const double groups = (double)((w.tiles_n + 3) / 4) * ((m + 15) / 16), products = (double)m * w.n * w.tiles_k * kW4TileK;
  return m <= 64 ||
         (bf16 ? 3.2 + 1.15e-3 * groups + 5.2e-9 * products : 4.0 + 2.0e-3 * groups + 10.5e-9 * products) <= tiles.us;
}

template <int kSteps, int kTerms, typename T>
hipError_t launch_tiles(const TilePlan& p, W4TileArgs a, hipStream_t stream) {
  a.tiles_m = (a.m + 16 * p.mt - 1) / (16 * p.mt);
  a.tiles_n = (a.w.tiles_n + 4 * p.nt - 1) / (4 * p.nt);
  const dim3 grid((unsigned)a.tiles_m * (unsigned)a.tiles_n);
#define TILES(NT, MT)                                                                               \
  if (p.nt == NT && p.mt == MT)                                                                     \
    hipLaunchKernelGGL((w4_tile_kernel<kSteps, NT, MT, kTerms, T>), grid, dim3(256), 0, stream, a);
  if constexpr (kTerms == 1) {
    TILES(2, 4) TILES(4, 4) TILES(3, 8)
  } else {
    TILES(2, 2) TILES(4, 2)
  }
#undef TILES
  return hipGetLastError();
}

// Whether the tiles' DMA takes rows of x as they lie.
template <typename X>
bool takes_rows(const void* x, uint32_t x_stride, int k) {
  return X::kTerms == 1 && k % 8 == 0 && x_stride % 8 == 0 && x_stride < kMaxTileStride && ((uintptr_t)x & 15u) == 0;
}

template <typename X>
hipError_t launch_many(const TilePlan& p, W4TileArgs a, const void* x, uint32_t x_stride, hipStream_t stream) {
  typedef typename X::Element T;
  a.k = a.w.k;
  if (takes_rows<X>(x, x_stride, a.w.k)) {
    a.x = static_cast<const uint16_t*>(x);
    a.ld = (int)x_stride;
  } else {
    a.k = a.ld = (a.w.k + 7) & ~7;
    a.plane = (size_t)a.m * (unsigned)a.ld;
    uint16_t* to = static_cast<uint16_t*>(staging(8, X::kTerms * a.plane * sizeof(uint16_t)));
    if (to == nullptr) return hipErrorOutOfMemory;
    const unsigned bx = (unsigned)(a.ld / 8 + 63) / 64;
    const unsigned by = std::min<unsigned>(((unsigned)a.m + 3) / 4, std::max(1u, 4096u / bx));
    hipLaunchKernelGGL((w4_terms_kernel<X>), dim3(bx, by), dim3(256), 0, stream, x, x_stride, to, a.plane, a.m, a.w.k,
                       a.ld);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.x = to;
  }
  switch (a.w.group) {
    case 32:
      return launch_tiles<4, X::kTerms, T>(p, a, stream);
    case 64:
      return launch_tiles<2, X::kTerms, T>(p, a, stream);
    default:
      return launch_tiles<1, X::kTerms, T>(p, a, stream);
  }
}

template <typename X>
hipError_t launch_few(W4Args a, hipStream_t stream) {
  RowsPlan p = plan_rows((uint32_t)a.m, a.w, X::kTerms == 1);
  if (p.slices > 1) {
    const size_t groups = (size_t)((a.w.tiles_n + p.nt - 1) / p.nt) * (unsigned)((a.m + 15) / 16);
    a.part = groups <= (size_t)kTickets
                 ? static_cast<float*>(staging(6, groups * (unsigned)p.slices * 256u * (unsigned)p.nt * sizeof(float)))
                 : nullptr;
    if (a.part == nullptr) p.slices = 1;
  }
  a.slices = p.slices;
  switch (a.w.group) {
    case 32:
      return launch_rows<X, 4>(p, a, stream);
    case 64:
      return launch_rows<X, 2>(p, a, stream);
    default:
      return launch_rows<X, 1>(p, a, stream);
  }
}

template <typename X>
hipError_t launch(const W4View& w, const void* x, uint32_t x_stride, void* out, uint32_t out_stride, uint32_t m,
                  hipStream_t stream) {
  constexpr bool kBf16 = X::kTerms == 1;
  const TilePlan p = plan_tiles(m, w, kBf16, !takes_rows<X>(x, x_stride, w.k));
  if (rows_are_few(m, w, kBf16, p)) return launch_few<X>(W4Args{w, x, out, nullptr, x_stride, out_stride, (int)m, 1}, stream);
  W4TileArgs a{};
  a.w = w;
  a.out = out;
  a.out_stride = out_stride;
  a.m = (int)m;
  return launch_many<X>(p, a, x, x_stride, stream);
}

}  // namespace

hipError_t launch_gemm_w4(const W4View& w, const void* x, uint32_t x_stride, void* out, uint32_t out_stride, bool bf16,
                          uint32_t m, hipStream_t stream) {
  return bf16 ? launch<W4RowsBf16>(w, x, x_stride, out, out_stride, m, stream)
              : launch<W4RowsF32>(w, x, x_stride, out, out_stride, m, stream);
}

}  // namespace prom
