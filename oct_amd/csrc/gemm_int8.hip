// The product of 8-bit rows: c[i, j] = a_scale[i] * w_scale[j] * sum_k a[i, k] w[j, k],
// a [m, k] and w [n, k] int8 with k contiguous in both, exact int32 sums.
//
// Two kernels.  Many rows: macro tiles on v_mfma_i32_32x32x32_i8.  A workgroup's
// waves form a kWM x kWN grid, each owning kMI x kNI blocks of 32 x 32.  Tiles of
// both operands (rows of 128 bytes of k, a whole line) travel HBM -> LDS by
// buffer_load ... lds into a ring of kSt stages; 16-byte chunks are XOR-swizzled by
// row, applied by each lane's source address, so that operand reads (16 bytes a
// lane, as they lie) are free of bank conflicts.  Descriptors end at the operand's
// end and a's chunks past k are sent out of range, so tails add zeros.  Rows that
// are not whole 16-byte chunks are copied to padded ones first.  Where tiles are few,
// K is cut into slices whose int32 sums a second kernel adds (exact in any order).
// 4224x20480x3840 to bf16: 328 to 343 us by the card, 2.03 to 1.94 POP/s (a library's product of the same shape to
// int32 308 to 345): five whole rounds of 256x256 tiles and the columns left over as
// 128x128 (as a sixth round 338).  Matrix units are busy 63 % of the time at a clock that
// their load lowers, waves wait 26 % of theirs, at the barrier of each K tile and for the first
// operands behind it.  Loads through registers instead of
// straight to LDS took 32 us longer, and at 4097x3001x513 to fp32 (5.7 us to pad and 22 for
// the tiles) saved no more than the padding cost.
//
// Few rows (a decode step, a short prompt): every weight is read once and K is dealt
// to the waves of a workgroup, which add their sums through LDS.  Bound by reading w:
// 1x32768x2048 12.3 us, 5.5 TB/s; 15x2048x16384 10.7 us.
#include <algorithm>
#include <type_traits>

#include "reactor_internal.h"

namespace prom {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kGroupM = 8;
constexpr uint32_t kOutOfRange = 0x80000000u;  // past every descriptor range

struct Int8Args {
  const int8_t* a;
  const int8_t* w;
  const float* a_scale;
  const float* w_scale;
  void* c;
  int32_t* slabs;  // K slices' sums, [slices][m][n] (null: one slice)
  int m, n, k;     // k of the operands as multiplied
  int lda, ldw, ldc;
  int tiles_m, tiles_n;
};

__device__ __forceinline__ void store_scaled(float* p, int sum, float as, float ws) { *p = (float)sum * as * ws; }
__device__ __forceinline__ void store_scaled(__bf16* p, int sum, float as, float ws) {
  *p = (__bf16)((float)sum * as * ws);
}

// 16 bytes of converted values from LDS words.
__device__ __forceinline__ void pack(const int32_t* from, int32_t (&to)[4]) {
  *reinterpret_cast<intx4*>(to) = *reinterpret_cast<const intx4*>(from);
}
__device__ __forceinline__ void pack(const int32_t* from, float (&to)[4]) {
  *reinterpret_cast<intx4*>(to) = *reinterpret_cast<const intx4*>(from);
}
__device__ __forceinline__ void pack(const int32_t* from, __bf16 (&to)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const intx4 v = *reinterpret_cast<const intx4*>(from + 4 * h);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[4 * h + i] = (__bf16)__int_as_float(v[i]);
  }
}

// 32 rows of kCols words in LDS (rows kPitch apart) to rows r0.. and columns c0.. of out [m, n], rows ld apart, 16
// bytes a lane at any alignment, the last columns of a row one by one.
template <int kCols, int kPitch, typename T>
__device__ __forceinline__ void store_rows(const int32_t* lds, T* out, int r0, int c0, int m, int n, int ld, int lane) {
  constexpr int kEach = 16 / (int)sizeof(T), kLanes = kCols / kEach, kRows = 64 / kLanes;
  const int c = (lane % kLanes) * kEach, left = n - (c0 + c);
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int r = i * kRows + lane / kLanes;
    if (r0 + r >= m || left <= 0) continue;
    T v[kEach];
    pack(lds + r * kPitch + c, v);
    T* to = out + (size_t)(r0 + r) * ld + c0 + c;
    if (left >= kEach) {
      __builtin_memcpy(to, v, 16);
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (j < left) to[j] = v[j];
    }
  }
}

template <int kMI_, int kNI_, int kWM_, int kWN_, int kSt_>
struct Cfg {
  static constexpr int kMI = kMI_, kNI = kNI_, kWM = kWM_, kWN = kWN_, kSt = kSt_, kBK = 128;
  static constexpr int kWaves = kWM * kWN;
  static constexpr int kBM = 32 * kMI * kWM, kBN = 32 * kNI * kWN;
  static constexpr int kABytes = kBM * kBK, kBBytes = kBN * kBK;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kAX = kABytes / 1024 / kWaves, kBX = kBBytes / 1024 / kWaves;  // transfers per wave and tile
  static constexpr int kX = kAX + kBX;
  static_assert(kAX * 1024 * kWaves == kABytes && kBX * 1024 * kWaves == kBBytes, "whole transfers per wave");
  static_assert(kSt >= 2 && kSt * kStage <= 163840 && (kSt - 2) * kX < 64, "ring");
};

// Position of chunk c of row r within the row's eight.
__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

template <int kN>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kN) : "memory");
}

// At most min(kMost, n) tiles of kX transfers may stay in flight.
template <int kX, int kMost>
__device__ __forceinline__ void wait_tiles(int n) {
  if constexpr (kMost > 0) {
    if (n < kMost) {
      wait_tiles<kX, kMost - 1>(n);
      return;
    }
  }
  wait_vmcnt<kX * kMost>();
}

template <class C, typename TOut>
__global__ __launch_bounds__(64 * C::kWaves, 2) void gemm_int8_tile_kernel(const Int8Args g) {
  __shared__ __attribute__((aligned(1024))) char lds[C::kSt * C::kStage];
  constexpr int kBK = C::kBK, kSteps = kBK / 32;
  const int num_tiles = g.tiles_m * g.tiles_n;
  int tm, tn;
  {
    const int pid = xcd_pid((int)blockIdx.x, num_tiles);
    const int per_group = kGroupM * g.tiles_n;
    const int group = pid / per_group;
    const int first_m = group * kGroupM;
    const int group_m = min(g.tiles_m - first_m, kGroupM);
    const int in_group = pid - group * per_group;
    tm = first_m + in_group % group_m;
    tn = in_group / group_m;
  }
  const int row0 = tm * C::kBM, col0 = tn * C::kBN;
  const int all_tiles = (g.k + kBK - 1) / kBK;
  const int slices = (int)gridDim.y;
  const int kt0 = (int)((long long)blockIdx.y * all_tiles / slices);
  const int kn = (int)((long long)(blockIdx.y + 1) * all_tiles / slices) - kt0;

  const int tid = (int)threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::kWN, wn = wave % C::kWN;

  // This wave's transfers: 1 KiB (eight rows) each.  Offsets are relative to the tile's first byte.
  uint32_t a_off[C::kAX], b_off[C::kBX];
  const int tr = lane >> 3;  // row within a transfer
#pragma unroll
  for (int i = 0; i < C::kAX; ++i) {
    const int r = 8 * (wave * C::kAX + i) + tr;
    a_off[i] = (uint32_t)(r * g.lda + 16 * ((lane & 7) ^ swz(r)));
  }
#pragma unroll
  for (int i = 0; i < C::kBX; ++i) {
    const int r = 8 * (wave * C::kBX + i) + tr;
    b_off[i] = (uint32_t)(r * g.ldw + 16 * ((lane & 7) ^ swz(r)));
  }
  const int k16 = (g.k + 15) & ~15;
  int issued = 0;
  // What is left of the tile's rows of each operand from the next k on (at most 256 rows of 2^17 bytes).
  const char* a_ptr = (const char*)(g.a + (size_t)row0 * g.lda + (size_t)kt0 * kBK);
  const char* b_ptr = (const char*)(g.w + (size_t)col0 * g.ldw + (size_t)kt0 * kBK);
  int a_left = (min(C::kBM, g.m - row0) - 1) * g.lda + k16 - kt0 * kBK;
  int b_left = (min(C::kBN, g.n - col0) - 1) * g.ldw + k16 - kt0 * kBK;
  auto desc = [](const char* p, int left) {
    const unsigned long long a = (unsigned long long)p;
    intx4 d;
    d.x = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffu));
    d.y = __builtin_amdgcn_readfirstlane((int)(a >> 32));
    d.z = __builtin_amdgcn_readfirstlane(left);
    d.w = 0x00020000;
    return d;
  };
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
  intx4 da = desc(a_ptr, a_left), db = desc(b_ptr, b_left);
  // LDS addresses of this wave's parts of the stage that the next tile goes to, and the stage's.
  uint32_t fill_a = __builtin_amdgcn_readfirstlane(lds0 + wave * C::kAX * 1024);
  uint32_t fill_b = __builtin_amdgcn_readfirstlane(lds0 + C::kABytes + wave * C::kBX * 1024);
  uint32_t fill_stage = 0;
  // Transfer j (0 .. kX-1) of the tile being issued; tail: a's last chunks lie past k.
  auto issue_one = [&](int j, bool tail) __attribute__((always_inline)) {
    if (j < C::kAX) {
      uint32_t off = a_off[j];
      if (tail) {
        const int r = 8 * (wave * C::kAX + j) + tr;
        if ((kt0 + issued) * kBK + 16 * ((lane & 7) ^ swz(r)) >= g.k) off = kOutOfRange;
      }
      const uint32_t to = __builtin_amdgcn_readfirstlane(fill_a + j * 1024);
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(da)
                   : "memory", "m0");
    } else {
      const uint32_t to = __builtin_amdgcn_readfirstlane(fill_b + (j - C::kAX) * 1024);
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(b_off[j - C::kAX]),
                   "s"(db)
                   : "memory", "m0");
    }
  };
  auto advance = [&]() __attribute__((always_inline)) {
    a_ptr += kBK;
    a_left -= kBK;
    b_ptr += kBK;
    b_left -= kBK;
    da = desc(a_ptr, a_left);
    db = desc(b_ptr, b_left);
    const bool round = fill_stage == (C::kSt - 1) * C::kStage;
    const uint32_t by = round ? 0u - (C::kSt - 1) * C::kStage : (uint32_t)C::kStage;
    fill_stage = round ? 0u : fill_stage + C::kStage;
    fill_a += by;
    fill_b += by;
    ++issued;
  };

  const int lrow = lane & 31;
  const int hk = lane >> 5;
  // Byte offsets within a stage: rows 32 further share the swizzle, and chunk 2 s + hk of a
  // row is chunk hk's position XOR 2 s, so mi and ni are immediate offsets of the reads.
  const int ra = wm * C::kMI * 32 + lrow, rb = wn * C::kNI * 32 + lrow;
  uint32_t a_base[kSteps], b_base[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    a_base[s] = (uint32_t)(ra * kBK + (((2 * s + hk) ^ swz(ra)) << 4));
    b_base[s] = (uint32_t)(C::kABytes + rb * kBK + (((2 * s + hk) ^ swz(rb)) << 4));
  }
  struct Frags {
    intx4 a[C::kMI], b[C::kNI];
  };
  auto read = [&](uint32_t st, int s) __attribute__((always_inline)) {
    Frags f;
    const char* pa = lds + (st + a_base[s]);
    const char* pb = lds + (st + b_base[s]);
#pragma unroll
    for (int mi = 0; mi < C::kMI; ++mi) f.a[mi] = *reinterpret_cast<const intx4*>(pa + mi * 32 * kBK);
#pragma unroll
    for (int ni = 0; ni < C::kNI; ++ni) f.b[ni] = *reinterpret_cast<const intx4*>(pb + ni * 32 * kBK);
    return f;
  };

  intx16 acc[C::kMI][C::kNI];
#pragma unroll
  for (int i = 0; i < C::kMI; ++i)
#pragma unroll
    for (int j = 0; j < C::kNI; ++j) acc[i][j] = intx16{};

  // The scales are fetched ahead of the sums: a thread a row's, a lane its columns'.
  float row_scale = 0.0f, ws[C::kNI];
  if (g.slabs == nullptr) {
    static_assert(C::kBM <= 64 * C::kWaves, "a thread a row");
    row_scale = g.a_scale[min(row0 + tid, g.m - 1)];
#pragma unroll
    for (int ni = 0; ni < C::kNI; ++ni) ws[ni] = g.w_scale[min(col0 + (wn * C::kNI + ni) * 32 + lrow, g.n - 1)];
  }

  // Tiles of this slice whose chunks of a all lie below k: all, or all but the last.
  const int whole = kn - ((kt0 + kn) * kBK > g.k ? 1 : 0);
#pragma unroll
  for (int s = 0; s < C::kSt - 1; ++s)
    if (s < kn) {
#pragma unroll
      for (int j = 0; j < C::kX; ++j) issue_one(j, s >= whole);
      advance();
    }
  constexpr int kDepth = C::kSt - 2;
  uint32_t cur = 0;
  // Step t: tile t has landed for this wave, later ones may stay in flight; after the
  // barrier it is complete for all waves and tile t-1's stage is free.  The transfers of
  // tile t + kSt - 1 go out between the MFMAs of the first half (4224x20480x3840: 338 us; over
  // all of them, where the last ones come late, 354, over a quarter 344).
  auto step = [&](int t, auto more_c, auto tail_c) __attribute__((always_inline)) {
    constexpr bool kMore = decltype(more_c)::value, kTail = decltype(tail_c)::value;
    constexpr int kMfma = kSteps * C::kMI * C::kNI;
    if constexpr (kMore && !kTail)
      wait_vmcnt<C::kX * kDepth>();
    else
      wait_tiles<C::kX, kDepth>(kn - 1 - t);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Frags f = read(cur, 0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Frags nf;
      if (s + 1 < kSteps) nf = read(cur, s + 1);
      __builtin_amdgcn_sched_barrier(0);  // the next step's reads go out before this one's MFMAs
#pragma unroll
      for (int mi = 0; mi < C::kMI; ++mi)
#pragma unroll
        for (int ni = 0; ni < C::kNI; ++ni) {
          const int at = (s * C::kMI + mi) * C::kNI + ni;
          acc[mi][ni] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[mi], f.b[ni], acc[mi][ni], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < C::kX; ++j)
            if (kMore && j * kMfma / C::kX / 2 == at) issue_one(j, kTail);
        }
      if (s + 1 < kSteps) f = nf;
    }
    if constexpr (kMore) advance();
    cur = cur + C::kStage == C::kSt * C::kStage ? 0 : cur + C::kStage;
  };
  const std::integral_constant<bool, true> yes{};
  const std::integral_constant<bool, false> no{};
  int t = 0;
  for (; t + C::kSt - 1 < whole; ++t) step(t, yes, no);
  if (t + C::kSt - 1 < kn) {
    step(t, yes, yes);
    ++t;
  }
  for (; t < kn; ++t) step(t, no, no);

  // Epilogue: 32 rows of the wave's columns at a time go through its part of LDS, so that a lane
  // stores 16 bytes of a row and neighbouring lanes neighbouring ones (stored from the accumulators,
  // two bytes a lane, 4224x20480 bf16 took 120 us longer).
  constexpr int kCols = 32 * C::kNI, kPitch = kCols + 4;
  static_assert((C::kWaves * 32 * kPitch + C::kBM) * 4 <= C::kSt * C::kStage, "the waves' parts and the scales");
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();  // the last tiles have been read
  asm volatile("" ::: "memory");
  int32_t* mine = reinterpret_cast<int32_t*>(lds) + wave * 32 * kPitch;
  float* scales = reinterpret_cast<float*>(lds) + C::kWaves * 32 * kPitch;
  if (g.slabs == nullptr) {
    if (tid < C::kBM) scales[tid] = row_scale;
    __syncthreads();
  }
  const int wave_col = col0 + wn * kCols;
#pragma unroll
  for (int mi = 0; mi < C::kMI; ++mi) {
    const int r0 = row0 + (wm * C::kMI + mi) * 32;
    if (r0 >= g.m) break;
    // Accumulator layout: lane l, register r holds row 8 (r/4) + 4 (l/32) + r%4, column l%32.
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dr = 8 * q + 4 * hk;
      const floatx4 as = *reinterpret_cast<const floatx4*>(scales + (wm * C::kMI + mi) * 32 + dr);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int ni = 0; ni < C::kNI; ++ni) {
          const int sum = acc[mi][ni][4 * q + r];
          mine[(dr + r) * kPitch + 32 * ni + lrow] =
              g.slabs == nullptr ? __float_as_int((float)sum * as[r] * ws[ni]) : sum;
        }
    }
    asm volatile("" ::: "memory");  // a wave's own part: its LDS operations stay in order
    if (g.slabs != nullptr)
      store_rows<kCols, kPitch>(mine, g.slabs + (size_t)blockIdx.y * g.m * g.n, r0, wave_col, g.m, g.n, g.n, lane);
    else
      store_rows<kCols, kPitch>(mine, static_cast<TOut*>(g.c), r0, wave_col, g.m, g.n, g.ldc, lane);
    asm volatile("" ::: "memory");
  }
}

// c = a_scale w_scale (sum of the K slices); the sums are exact, whatever their order.
template <typename TOut>
__global__ __launch_bounds__(256) void int8_slices_kernel(const int32_t* __restrict__ slabs, int slices,
                                                          const float* __restrict__ a_scale,
                                                          const float* __restrict__ w_scale, TOut* __restrict__ c,
                                                          int m, int n, int ldc) {
  const int col = (int)(blockIdx.x * 256 + threadIdx.x);
  if (col >= n) return;
  const size_t slab = (size_t)m * n;
  const float ws = w_scale[col];
  for (int row = (int)blockIdx.y; row < m; row += (int)gridDim.y) {
    const int32_t* p = slabs + (size_t)row * n + col;
    int sum = 0;
    for (int s = 0; s < slices; ++s) sum += p[s * slab];
    store_scaled(c + (size_t)row * ldc + col, sum, a_scale[row], ws);
  }
}

// Sixteen bytes from column k of a row at any alignment, zeros from column `cols` on: the row's last
// sixteen, shifted, where it ends within them.
__device__ __forceinline__ intx4 load16(const int8_t* row, int k, int cols) {
  intx4 v = {0, 0, 0, 0};
  const int past = k + 16 - cols;
  if (past <= 0) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (past < 16 && cols >= 16) {
    unsigned __int128 b;
    __builtin_memcpy(&b, row + cols - 16, 16);
    b >>= 8 * past;
    __builtin_memcpy(&v, &b, 16);
  } else if (past < 16) {
    int8_t b[16] = {};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < cols) b[j] = row[k + j];
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

// Both operands' rows, cols bytes each, to rows of ld (a multiple of 16), zero from column cols on:
// sixteen bytes a thread, read at any alignment.
__global__ __launch_bounds__(256) void pad_rows8_kernel(const int8_t* __restrict__ a, int8_t* __restrict__ to_a, int m,
                                                        const int8_t* __restrict__ w, int8_t* __restrict__ to_w, int n,
                                                        int cols, int ld) {
  const int chunks = ld / 16;
  const long long total = ((long long)m + n) * chunks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int row = (int)(i / chunks), c = (int)(i - (long long)row * chunks) * 16;
    const bool first = row < m;
    const size_t r = (size_t)(first ? row : row - m);
    const intx4 v = load16((first ? a : w) + r * cols, c, cols);
    *reinterpret_cast<intx4*>((first ? to_a : to_w) + r * ld + c) = v;
  }
}

// Few rows: a workgroup computes 16 columns of c for 16 kMT rows; its waves take K in turn, 256 bytes
// of every row at a time, the next step's loads out while one is multiplied.  The matrix instruction
// wants another row in each of 16 neighbouring lanes, a load neighbouring bytes there (loaded as they
// are multiplied, a load keeps the cache four times as long: 15x2048x16384 16.4 us, now 8.6).  So a
// load takes 256 bytes of four rows, and the wave's own part of LDS turns them, 16-byte chunks XORed
// by row against bank conflicts.
template <int kMT, int kWaves, typename TOut>
__global__ __launch_bounds__(64 * kWaves) void gemm_int8_rows_kernel(const Int8Args g) {
  constexpr int kSeg = 256, kWLoads = 4, kALoads = 4 * kMT, kBytes = 1024 * (kWLoads + kALoads);
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kBytes];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r16 = lane & 15, h = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * kMT;
  char* lw = lds + wave * kBytes;
  char* la = lw + 1024 * kWLoads;
  struct Step {
    intx4 w[kWLoads], a[kALoads];
  };
  auto load = [&](Step& s, int t, auto tail_c) __attribute__((always_inline)) {
    constexpr bool kTail = decltype(tail_c)::value;
    const int k = t * kSeg + 16 * r16;
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) {
      const int8_t* p = g.w + (size_t)min(n0 + 4 * i + h, g.n - 1) * g.k;
      if constexpr (kTail)
        s.w[i] = load16(p, k, g.k);
      else
        __builtin_memcpy(&s.w[i], p + k, 16);
    }
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const int row = m0 + 4 * i + h;
      s.a[i] = intx4{0, 0, 0, 0};
      if (row >= g.m) continue;
      const int8_t* p = g.a + (size_t)row * g.k;
      if constexpr (kTail)
        s.a[i] = load16(p, k, g.k);
      else
        __builtin_memcpy(&s.a[i], p + k, 16);
    }
  };
  auto put = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) {
      const int r = 4 * i + h;
      *reinterpret_cast<intx4*>(lw + r * kSeg + ((r16 ^ (r & 15)) << 4)) = s.w[i];
    }
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const int r = 4 * i + h;
      *reinterpret_cast<intx4*>(la + r * kSeg + ((r16 ^ (r & 15)) << 4)) = s.a[i];
    }
  };
  intx4 acc[kMT] = {};
  auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = r16 * kSeg + (((4 * u + h) ^ r16) << 4);
      const intx4 w = *reinterpret_cast<const intx4*>(lw + at);
#pragma unroll
      for (int i = 0; i < kMT; ++i)
        acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, *reinterpret_cast<const intx4*>(la + 16 * i * kSeg + at),
                                                       acc[i], 0, 0, 0);
    }
  };
  // The wave's own part: its LDS operations stay in order.
  auto fence = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  };
  const std::integral_constant<bool, true> yes{};
  const std::integral_constant<bool, false> no{};
  const int whole = g.k / kSeg;  // steps without a tail
  int t = wave;
  if (t < whole) {
    Step s;
    load(s, t, no);
    for (; t + kWaves < whole; t += kWaves) {
      put(s);
      load(s, t + kWaves, no);
      fence();
      multiply();
      fence();
    }
    put(s);
    fence();
    multiply();
    fence();
  }
  if (whole * kSeg < g.k && whole % kWaves == wave) {
    Step s;
    load(s, whole, yes);
    put(s);
    fence();
    multiply();
  }
  __syncthreads();  // the operands have been read
  intx4* part = reinterpret_cast<intx4*>(lds) + lane;  // [wave - 1][kMT][64]
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < kMT; ++i) part[((wave - 1) * kMT + i) * 64] = acc[i];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int s = 0; s < kWaves - 1; ++s)
#pragma unroll
    for (int i = 0; i < kMT; ++i) acc[i] += part[(s * kMT + i) * 64];
  // Lane l, register r: column (of w) 4 (l/16) + r, row (of a) l%16.
#pragma unroll
  for (int i = 0; i < kMT; ++i) {
    const int row = m0 + 16 * i + r16;
    if (row >= g.m) continue;
    const float as = g.a_scale[row];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int col = n0 + 4 * h + r;
      if (col < g.n) store_scaled(static_cast<TOut*>(g.c) + (size_t)row * g.ldc + col, acc[i][r], as, g.w_scale[col]);
    }
  }
}

#define INT8_TILES(X)               \
  X(0, 1, 1, 2, 2, 4) /* 64x64 */   \
  X(1, 1, 2, 4, 2, 4) /* 128x128 */ \
  X(2, 2, 2, 2, 2, 2) /* 128x128, two workgroups a CU */ \
  X(3, 3, 2, 2, 4, 2) /* 192x256 */ \
  X(4, 4, 2, 2, 4, 2) /* 256x256 */

struct TileInfo {
  int bm, bn, threads;
};
#define X(i, ...) {Cfg<__VA_ARGS__>::kBM, Cfg<__VA_ARGS__>::kBN, 64 * Cfg<__VA_ARGS__>::kWaves},
constexpr TileInfo kTiles[] = {INT8_TILES(X)};
#undef X
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);

template <typename TOut>
hipError_t launch_tile(int tile, int slices, const Int8Args& g, hipStream_t stream) {
  const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), (unsigned)slices);
  const dim3 block((unsigned)kTiles[tile].threads);
  switch (tile) {
#define X(i, ...)                                                                                    \
  case i:                                                                                            \
    hipLaunchKernelGGL((gemm_int8_tile_kernel<Cfg<__VA_ARGS__>, TOut>), grid, block, 0, stream, g);  \
    break;
    INT8_TILES(X)
#undef X
  }
  return hipGetLastError();
}

// Estimated microseconds of a tile's workgroup: `fill` plus step[w - 1] for each 128 of k where w of
// them share a CU; on an otherwise idle chip a step takes `idle` of that.  From 15 x 17 tiles of
// each with k 512, 2048 and 8192, two and three rounds of them, and a single tile.
struct TileCost {
  int occ;
  double step[2], fill, idle;
};
constexpr TileCost kCost[kNumTiles] = {
    {2, {0.215, 0.46}, 2.3, 0.95},  // 64x64
    {1, {0.615, 0.0}, 4.3, 0.73},   // 128x128
    {2, {0.72, 1.16}, 3.1, 0.54},   // 128x128, two a CU
    {1, {1.45, 0.0}, 8.3, 0.54},    // 192x256
    {1, {1.60, 0.0}, 12.5, 0.60},   // 256x256
};
constexpr double kLaunchUs = 3.0;  // of a further launch

double rounds_us(int t, uint64_t workgroups, uint32_t kt) {
  const TileCost& c = kCost[t];
  const uint64_t full = c.occ == 2 ? workgroups >> 9 : workgroups >> 8;
  const uint32_t rest = (uint32_t)(workgroups - full * 256 * (uint64_t)c.occ);
  double us = (double)full * (c.fill + kt * c.step[c.occ - 1]);
  if (rest > 0) {
    const uint32_t w = (rest + 255) >> 8;
    us += c.fill + kt * c.step[w - 1] * (c.idle + (1.0 - c.idle) / 256.0 * rest / w);
  }
  return us;
}

struct Plan {
  int tile, slices;
  uint32_t n;  // columns that it takes
};
uint64_t tiles_of(int t, uint32_t m, uint32_t n) {
  const uint32_t bm = (uint32_t)kTiles[t].bm, bn = (uint32_t)kTiles[t].bn;
  return (uint64_t)((m + bm - 1) / bm) * ((n + bn - 1) / bn);
}
// The best tile and number of K slices for all of n columns; slices where tiles are no two rounds.
double plan_columns(uint32_t m, uint32_t n, uint32_t k, Plan* plan) {
  static const uint32_t kSlices[] = {1, 2, 3, 4, 6, 8, 12, 16};
  const uint32_t all = (k + 127) / 128;
  double best = 1e300;
  for (int t = 0; t < kNumTiles; ++t) {
    const uint64_t tiles = tiles_of(t, m, n);
    for (uint32_t s : kSlices) {
      if (s > 1 && (all < 3 * s || tiles >= 512u * (unsigned)kCost[t].occ)) break;
      double us = rounds_us(t, tiles * s, (all + s - 1) / s);
      if (s > 1) us += 6.1 + (double)(s + 1) * m * n * 4.0 / 10.0e6;
      if (us < best) {
        best = us;
        *plan = Plan{t, (int)s, n};
      }
    }
  }
  return best;
}
// Or one tile for as many columns as are whole rounds of it, and another plan for the rest, where that
// promises 3 % (estimates are not that good).
int plan_tiles(uint32_t m, uint32_t n, uint32_t k, Plan (&plan)[2]) {
  double best = 0.97 * plan_columns(m, n, k, &plan[0]);
  int parts = 1;
  for (int t = 1; t < kNumTiles; ++t) {
    const uint64_t tiles = tiles_of(t, m, n), slots = 256u * (unsigned)kCost[t].occ;
    if (tiles <= slots) continue;
    const uint64_t columns = tiles / slots * slots / tiles_of(t, m, 1) * (unsigned)kTiles[t].bn;
    if (columns == 0 || columns >= n) continue;
    Plan rest;
    const double us = rounds_us(t, tiles_of(t, m, (uint32_t)columns), (k + 127) / 128) + kLaunchUs +
                      plan_columns(m, n - (uint32_t)columns, k, &rest);
    if (us < best) {
      best = us;
      parts = 2;
      plan[0] = Plan{t, 1, (uint32_t)columns};
      plan[1] = rest;
    }
  }
  return parts;
}

template <typename TOut>
hipError_t launch_rows(Int8Args g, hipStream_t stream) {
#define ROWS(MT, W)                                                                          \
  hipLaunchKernelGGL((gemm_int8_rows_kernel<MT, W, TOut>), dim3((unsigned)((g.n + 15) / 16), \
                     (unsigned)((g.m + 16 * MT - 1) / (16 * MT))), dim3(64 * W), 0, stream, g)
  // More waves a workgroup where it has a long K to itself (us with 4, 8, 16 waves: 1x8192x2048 4.7, 5.3,
  // 5.6; 1x12288x4096 9.4, 10.6, 12.1; 1x2048x8192 6.0, 5.3, 5.5; 15x2048x16384 -, 11.8, 10.7; 16x2048x65536
  // 38, 28, 27; 16 do not fit LDS with 32 rows).
  const int waves = g.n >= 16 * 1024 || g.k <= 4096 ? 4 : g.m > 16 || g.n > 4096 || g.k <= 8192 ? 8 : 16;
  // A launch has fewer than 2^32 threads: more than 2^27 columns (four waves take 16) go in blocks.
  for (int left = g.n; left > 0; left -= g.n) {
    g.n = std::min(left, 1 << 27);
    if (g.m > 16) {
      if (waves == 4)
        ROWS(2, 4);
      else
        ROWS(2, 8);
    } else if (waves == 4) {
      ROWS(1, 4);
    } else if (waves == 8) {
      ROWS(1, 8);
    } else {
      ROWS(1, 16);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    g.w += (size_t)g.n * g.k;
    g.w_scale += g.n;
    g.c = static_cast<TOut*>(g.c) + g.n;
  }
#undef ROWS
  return hipSuccess;
}

constexpr uint32_t kFewRows = 32;

template <typename TOut>
hipError_t launch(Int8Args g, hipStream_t stream) {
  const uint32_t m = (uint32_t)g.m, n = (uint32_t)g.n, k = (uint32_t)g.k;
  g.ldc = g.n;
  if (m <= kFewRows) return launch_rows<TOut>(g, stream);
  g.lda = g.ldw = g.k;
  const bool aligned = k % 16 == 0 && ((uintptr_t)g.a & 15u) == 0 && ((uintptr_t)g.w & 15u) == 0;
  if (!aligned) {
    const int ld = (int)((k + 15) & ~15u);
    int8_t* pa = static_cast<int8_t*>(staging(8, (size_t)m * ld));
    int8_t* pw = static_cast<int8_t*>(staging(9, (size_t)n * ld));
    if (pa == nullptr || pw == nullptr) return hipErrorOutOfMemory;
    const unsigned long long chunks = ((unsigned long long)m + n) * (unsigned)(ld / 16);
    hipLaunchKernelGGL(pad_rows8_kernel, dim3((unsigned)std::min<unsigned long long>((chunks + 255) / 256, 1u << 16)),
                       dim3(256), 0, stream, g.a, pa, g.m, g.w, pw, g.n, g.k, ld);
    g.a = pa;
    g.w = pw;
    g.lda = g.ldw = ld;
  }
  Plan plans[2];
  const int parts = plan_tiles(m, n, k, plans);
  for (int i = 0; i < parts; ++i) {
    Plan& p = plans[i];
    g.n = (int)p.n;
    g.slabs = nullptr;
    if (p.slices > 1) {
      g.slabs = static_cast<int32_t*>(staging(6, (size_t)p.slices * m * p.n * sizeof(int32_t)));
      if (g.slabs == nullptr) p.slices = 1;
    }
    g.tiles_m = (int)((m + kTiles[p.tile].bm - 1) / kTiles[p.tile].bm);
    g.tiles_n = (int)((p.n + kTiles[p.tile].bn - 1) / kTiles[p.tile].bn);
    const hipError_t e = launch_tile<TOut>(p.tile, p.slices, g, stream);
    if (e != hipSuccess) return e;
    if (p.slices > 1)
      hipLaunchKernelGGL((int8_slices_kernel<TOut>), dim3((p.n + 255) / 256, std::min<unsigned>(m, 4096u)), dim3(256),
                         0, stream, g.slabs, p.slices, g.a_scale, g.w_scale, static_cast<TOut*>(g.c), g.m, g.n, g.ldc);
    g.w += (size_t)p.n * g.ldw;
    g.w_scale += p.n;
    g.c = static_cast<TOut*>(g.c) + p.n;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gemm_int8(const int8_t* a, const int8_t* w, const float* a_scale, const float* w_scale, void* c,
                            bool bf16, uint32_t m, uint32_t n, uint32_t k, hipStream_t stream) {
  Int8Args g{};
  g.a = a;
  g.w = w;
  g.a_scale = a_scale;
  g.w_scale = w_scale;
  g.c = c;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  return bf16 ? launch<__bf16>(g, stream) : launch<float>(g, stream);
}

}  // namespace prom
