// Products of ragged groups of columns on the sm_100a tensor cores (Float16 / BFloat16), run sizes on the device:
//
//     C[:, i] = A_g X[:, columns[i]]            for the columns i of run g
//             + B_a T[:, i]                     for low-rank pairs, T = scale * A_a X in two 16-bit terms
//
// The tensor core computes D[m, i] = sum_k P[m, k] Q[i, k]: rows of a matrix in the 128 lanes of tensor memory, a run's
// columns along its columns.  That way round a tile's number of columns can be any multiple of 16 (the instruction's N is its own), so
// that a run of 300 is two tiles of 160 and 140 and not 256 and 44, and one of 3 is padded to 16 and not to 128.
//
// A CTA owns a tile of 128 rows x at most NT columns, a pair of CTAs (cta_group::2) one of 256 x 256, and walks over K in blocks of 64; the
// grid is persistent.
//   prologue    every CTA counts the tiles of all runs (at most kMaxRuns) into a table in shared memory
//   warps 0, 10, 11  TMA producers, every third stage each: a ring of stages, each a K block (of a pair two) of the matrix (K- or MN-major,
//               as it is stored) and of the columns (K-major); gathered columns arrive four at a time (tile::gather4), their numbers in
//               the lanes' registers.  One thread takes some 125 cycles for a copy: with a single producer a stage took 765 cycles,
//               148 of them 4.2 TB/s
//   warp 1      allocates tensor memory, issues every tcgen05.mma; a low-rank pair's are of the 16 columns (PAIR: 32) that its runs are in, where
//               it first clears the rows of T that belong to other runs
//   warps 2-9   epilogue: tensor memory -> registers -> shared memory, transposed -> C
// A matrix B_a with infinities or NaN may meet neither those cleared rows nor the second terms of T, which can have the other sign: zero times
// infinity, and infinity minus infinity, would be NaN in columns of other requests and in its own.  So the product A X, whose epilogue has
// nothing to do at first, looks through the B_a in use and leaves a byte for each 128 rows of each, and where one is set the pair is
// added by the epilogue in Float32.  (6160 columns in 8 runs, 4096 x 4096, rank 64: 194 us; 205 where the issuing warp looks through the blocks as they arrive.)
// Two accumulators alternate, so that the epilogue of one tile overlaps the products of the next.
//
// What bounds it: reading the matrices while a run is a few columns (128 experts of 1536 x 2048, 32 tokens of 8 each: 100 us, 1.2 of what reading those
// in use takes at 6.55 TB/s), the tensor cores under the power limit where it is hundreds (8192 tokens twice: 1361 us, 1413 TFLOP/s).
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "common.cuh"
#include "early.cuh"
#include "grouped_runs.cuh"
#include "launchers.h"
#include "umma.cuh"
#include "umma_shared.cuh"

namespace nb200 {

__device__ int g_grouped_abort = 0;  // sticky: a bounded wait of one of these kernels ran out

namespace {

constexpr int kThreads = 384;
constexpr int kProducers = 3;              // warps 0, 10, 11: a copy costs its thread some 125 cycles, a stage has up to eight
constexpr int kBK = 64;                  // K elements per stage: one 128-byte swizzle row
constexpr int kHalfBytes = 128 * 128;    // 128 rows x 64 K elements, either layout
constexpr int kMaxRuns = 1024;
constexpr int kAhead = 8;                // column tiles that a band of row tiles shares
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);   // 8-row groups 1024 bytes apart, 128-byte swizzle

// Runs in shared memory: the product's own where they have offsets (column tiles of the runs before run i, its first column, the column
// behind it), else those of low-rank pairs (cum: the pair).  From global memory a tile's search for its pairs took 7000 cycles.
struct Table {
  int cum[kMaxRuns + 8], begin[kMaxRuns], end[kMaxRuns];
};
constexpr int kTableBytes = sizeof(Table);
constexpr int kOutBytes = 8 * 2048;      // a box of 32 rows x 32 columns for each warp of the epilogue

// PAIR: two CTAs of a cluster on one tile, 128 rows and half of the columns' operand each
template <int NT, bool PAIR>
struct Cfg {
  // K blocks of 64 in a stage: a wait, a commit and a turn of the loop took the issuing thread 370 cycles, a pair's products of a block 512
  static constexpr int kSub = PAIR ? 2 : 1;
  static constexpr int kA = kHalfBytes, kX = NT * 128 / (PAIR ? 2 : 1), kXOff = kSub * kA, kStage = kSub * (kA + kX);
  static constexpr int kRoom = 226 * 1024 - kTableBytes - kOutBytes - 512;
  static constexpr int kStages = kRoom / kStage > 10 ? 10 : kRoom / kStage;
  static constexpr int kTmemCols = 2 * NT;               // two accumulators
  static constexpr int kBox = NT >= 128 ? 64 : 16;       // columns of X that one copy brings
  static constexpr int kOutOff = kStages * kStage, kTableOff = kOutOff + kOutBytes, kBarOff = kTableOff + kTableBytes;
  static constexpr int kSmem = kBarOff + 512 + 1024;
};
static_assert(Cfg<256, true>::kStages == 3 && Cfg<256, false>::kStages == 4 && Cfg<32, false>::kStages == 9, "ring depth");
static_assert(Cfg<256, true>::kSmem <= 232448 && Cfg<256, false>::kSmem <= 232448 && Cfg<128, false>::kSmem <= 232448 && Cfg<64, false>::kSmem <= 232448 &&
              Cfg<32, false>::kSmem <= 232448, "shared memory budget");

struct Bars {
  uint64_t full[10], empty[10], acc_full[2], acc_empty[2];
  uint64_t side[6];                      // PAIR, stages of which columns are to be cleared: the second CTA's copies are there; in the first CTA: are cleared
  uint32_t tmem_base;
  int abort_flag;
  int odd;                               // sticky: a pair was left to the epilogue
  RunSearch search;
};
static_assert(sizeof(Bars) <= 512, "barrier block");

enum { kToC, kToParts, kToLow };         // what the epilogue writes
enum { kWaitNone, kWaitData, kWaitEnd }; // launched early: what the kernel before writes is read from the start, or not at all

struct FwdArgs {
  Runs runs;
  const int* ids;
  const int* columns;
  void* C;                               // kToParts: Float32 (M, R, splits); kToLow: T, 16-bit
  long long ldc;
  const float* scale;
  float scale0;
  int M, K, G, N, mats;
  int cap;                               // columns of a tile, at most NT
  int a_kmaj, a_same, zero_rest, splits, tiles_m, to, vec, gather;
  int low_width, low_step;               // elements of T for a column, of each of its terms
  Runs low_runs;                         // kToC: low-rank pairs, r = 0: none
  const int* low_ids;
  const void* low_B;                     // as the caller has it
  long long low_ldb, low_strideB;
  const void* low_T;
  unsigned char* odd;                    // (n, 128s of rows of B): whether there are infinities or NaN; read, or, look_r > 0, found out
  int look_r, look_m;                    // rank of B, its rows
  int r, n, low_kmaj, low_same;          // same: one matrix for all pairs
  int wait;
  int* status;
};

// four rows of a 2-d tensor map, 64 elements each
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | ((uint32_t)((kHalfBytes / 2) >> 4) << 16); }
// ---- two CTAs as one
__device__ __forceinline__ int cluster_rank() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// an arrival at the first CTA's barrier
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
}
// copies of a pair: their bytes count at the first CTA's barrier, whose address this is in the cluster
__device__ __forceinline__ uint32_t first_barrier(uint64_t* bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
  return a;
}
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void pair_load_3d(void* dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// mbar_wait for a barrier that the other CTA arrives at
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  auto look = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
  };
#pragma unroll 1
  for (int it = 0; it < 4096; ++it)
    if (look()) return true;
  const unsigned long long t0 = globaltimer_ns();
#pragma unroll 1
  while (true) {
#pragma unroll 1
    for (int it = 0; it < 32; ++it)
      if (look()) return true;
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      return false;
    }
  }
}
template <bool PAIR>
__device__ __forceinline__ bool wait_of(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, PAIR ? wait_cluster(bar, parity, abort_flag) : mbar_wait(bar, parity, abort_flag)) != 0;
}
// One thread's instructions, called by a whole warp in step: what they take is then computed in uniform registers, where the instruction
// wants it.
template <bool PAIR>
__device__ __forceinline__ void multiply_add(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
#define NB_MMA(GROUP)                                                                                    \
  asm volatile(                                                                                          \
      "{\n\t"                                                                                            \
      ".reg .pred p, one;\n\t"                                                                           \
      ".reg .b64 da, db;\n\t"                                                                            \
      "mov.b64 da, {%1, %3};\n\t"                                                                        \
      "mov.b64 db, {%2, %3};\n\t"                                                                        \
      "setp.ne.b32 p, %5, 0;\n\t"                                                                        \
      "elect.sync _|one, 0xffffffff;\n\t"                                                                \
      "@one tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, p;\n\t"                         \
      "}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)                      \
      : "memory")
  if constexpr (PAIR) NB_MMA("2");
  else NB_MMA("1");
#undef NB_MMA
}
// an arrival (PAIR: at both CTAs' barriers) when what was issued so far has completed
template <bool PAIR>
__device__ __forceinline__ void commit_to(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t"
        "}" ::"r"(smem_u32(bar)), "h"((unsigned short)3)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}" ::"r"(smem_u32(bar))
        : "memory");
}
// a wait of a warp in step
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}
template <bool PAIR>
__device__ __forceinline__ void take_tmem(uint32_t* result, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(result)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(result, columns);
    tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void give_tmem(uint32_t addr, uint32_t columns) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else tmem_dealloc(addr, columns);
}
template <bool PAIR>
__device__ __forceinline__ void sync_all() {
  if constexpr (PAIR) {
    __syncwarp();
    cluster_sync();
  } else {
    __syncthreads();
  }
}
// barriers, tensor memory and the abort flag of a CTA; the whole block's
template <int NT, bool PAIR>
__device__ __forceinline__ void set_up(Bars* bars) {
  using C = Cfg<NT, PAIR>;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
      if (PAIR) mbar_init(&bars->side[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->acc_full[s], 1);
      mbar_init(&bars->acc_empty[s], PAIR ? 16 : 8);
    }
    bars->abort_flag = *reinterpret_cast<volatile int*>(&g_grouped_abort);
    bars->odd = 0;
    fence_mbar_init();
  }
  if ((threadIdx.x >> 5) == 1) take_tmem<PAIR>(&bars->tmem_base, C::kTmemCols);
}
template <int NT, bool PAIR>
__device__ __forceinline__ void tear_down(Bars* bars, uint32_t tmem, int* status) {
  tc_fence_before();
  sync_all<PAIR>();                                       // (the first CTA's products read the other's shared memory)
  if ((threadIdx.x >> 5) == 1) {
    tc_fence_after();
    give_tmem<PAIR>(tmem, Cfg<NT, PAIR>::kTmemCols);
  }
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int*>(&bars->abort_flag)) {
    atomicExch(&g_grouped_abort, 1);
    if (status) atomicExch(status, NNLIB_B200_TIMEOUT);
  }
  sync_all<PAIR>();
}
template <bool PAIR>
__device__ __forceinline__ uint32_t idesc_of(bool bf16, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
}
// T of a column is kept as two terms of 16 bits, together 16 (BFloat16) or 22 bits of it: one alone would be off by what the result is rounded by.
// Float16 has no such bits below 2^-14: what is left of a T of 1e-4 is off by 1.7e-4 of T, of 1e-6 by 2 %.  A product is so off by at most 2^-25
// times the magnitudes in a row of B, where its own result's smallest steps are 2^-24; but the gradients add up many such T.  They take the second
// term 2^11 times as large, from a third place (at most 2^15: what is left of the largest numbers is 2^4): its step is 2^-35.
// Nothing is left of what is infinite: Inf - Inf would be a NaN.
constexpr float kScaled = 2048.f;
template <typename T>
__device__ __forceinline__ void put_terms(T* out, int step, float v) {
  const T first = Elem<T>::from_f(v);
  const float left = fabsf(Elem<T>::to_f(first)) < INFINITY ? v - Elem<T>::to_f(first) : 0.f;
  constexpr bool kThree = std::is_same<T, __half>::value;
  out[kThree ? step : 0] = first;
  out[kThree ? 0 : step] = Elem<T>::from_f(left);
  if constexpr (kThree) out[2 * step] = Elem<T>::from_f(left * kScaled);
}
// A gradient's sum from those of the first and the second terms.  A first that is infinite met an infinity of the other array, whose product with the second
// term, a zero or of the other sign, would make a NaN of it.
__device__ __forceinline__ float both_terms(uint32_t first, uint32_t second, float scale) {
  const float v = fmaf(scale, __uint_as_float(second), __uint_as_float(first));
  float r;
  asm("{\n\t.reg .pred p;\n\tsetp.nan.f32 p, %1, %1;\n\tselp.f32 %0, %2, %1, p;\n\t}" : "=f"(r) : "f"(v), "f"(__uint_as_float(first)));
  return r;
}
__device__ __forceinline__ int round16(int n) { return (n + 15) & ~15; }
// columns that a product takes are so many at a time (PAIR: half of them from each CTA)
template <bool PAIR> constexpr int kGrain = PAIR ? 32 : 16;
template <bool PAIR>
__device__ __forceinline__ int product_columns(int n) { return (n + kGrain<PAIR> - 1) & ~(kGrain<PAIR> - 1); }

// Width of the tiles of a run of n columns, and their number: at most cap (a multiple of 16) and as even as multiples of 16 allow.
__host__ __device__ __forceinline__ int tile_width(int n, int cap) {
  const int c = (n + cap - 1) / cap;
  return c > 0 ? ((n + c - 1) / c + 15) & ~15 : 16;
}
__host__ __device__ __forceinline__ int tile_count(int n, int cap) {
  const int w = tile_width(n, cap);
  return (n + w - 1) / w;
}

// Fills the table (runs of one length need none).  By the whole block.  Whether offsets fall somewhere.
__device__ bool count_tiles(const FwdArgs& g, Table& tab, RunSearch& s) {
  if (!g.runs.offsets) {
    if (g.r == 0 || g.low_runs.runs > kMaxRuns) return false;          // (more have no offsets)
    bool falls = false;
    for (int i = threadIdx.x; i < g.low_runs.runs; i += kThreads) {
      tab.cum[i] = g.low_ids[i];
      tab.begin[i] = g.low_runs.begin(i);
      tab.end[i] = g.low_runs.end(i);
      falls = falls || g.low_runs.at(i + 1) < g.low_runs.at(i);
    }
    return __syncthreads_or(falls) != 0;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int carry = 0;
  bool falls = false;
  for (int i0 = 0; i0 < g.G; i0 += kThreads) {
    const int i = i0 + (int)threadIdx.x;
    int own = 0;
    if (i < g.G) {
      const int mat = g.ids ? g.ids[i] : i, begin = g.runs.begin(i), end = g.runs.end(i);
      if (mat >= 0 && mat < g.mats) own = tile_count(end - begin, g.cap);
      tab.begin[i] = begin;
      tab.end[i] = end;
      falls = falls || g.runs.at(i + 1) < begin;
    }
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (lane == 31) s.part[warp] = sum;
    __syncthreads();
    int before = carry, all = carry;
    for (int q = 0; q < kThreads / 32; ++q) {
      if (q < warp) before += s.part[q];
      all += s.part[q];
    }
    if (i < g.G) tab.cum[i] = before + sum - own;
    carry = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) tab.cum[g.G] = carry;
  return __syncthreads_or(falls) != 0;
}

// Place in a ring of N stages: no divisions, which cost as much as a stage's copies do.
template <int N>
struct Ring {
  int s = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) { s = 0; ++round; }
  }
  __device__ __forceinline__ void skip(int n) {
    s += n;
    round += s / N;
    s %= N;
  }
};

struct Tile {
  int run, mat, n0, nt, m0, kb0, kb1, split;
};
template <bool PAIR>
__device__ __forceinline__ Tile tile_of(const FwdArgs& g, const Table& tab, long long t, int nkb) {
  Tile o;
  o.split = (int)(t % g.splits);
  const long long q = t / g.splits;
  int tiles, run, begin, end;
  long long at;
  if (g.runs.offsets) {
    const int col = (int)(q / g.tiles_m);                  // the last run with cum[run] <= col
    int lo = 0, hi = g.G;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tab.cum[mid] <= col) lo = mid; else hi = mid;
    }
    run = lo;
    tiles = tab.cum[run + 1] - tab.cum[run];
    at = q - (long long)tab.cum[run] * g.tiles_m;
    begin = tab.begin[run];
    end = tab.end[run];
  } else {
    tiles = tile_count((int)g.runs.len, g.cap);
    run = (int)(q / ((long long)tiles * g.tiles_m));
    at = q - (long long)run * tiles * g.tiles_m;
    begin = g.runs.begin(run);
    end = g.runs.end(run);
  }
  // bands of kAhead column tiles: what runs at the same time shares the matrix's rows and the columns
  const int band = (int)(at / (kAhead * g.tiles_m)), in = (int)(at - (long long)band * kAhead * g.tiles_m), wide = min(kAhead, tiles - band * kAhead);
  const int w = tile_width(end - begin, g.cap);
  o.run = run;
  o.mat = g.ids ? g.ids[run] : run;
  o.m0 = (in / wide) * (PAIR ? 256 : 128);
  o.n0 = begin + (band * kAhead + in % wide) * w;
  o.nt = o.mat >= 0 && o.mat < g.mats ? min(w, end - o.n0) : 0;      // (0: nothing to do)
  o.kb0 = (int)((long long)nkb * o.split / g.splits);
  o.kb1 = (int)((long long)nkb * (o.split + 1) / g.splits);
  return o;
}

// Runs of low-rank pairs that have columns in a tile, neighbours of the same pair as one.  Where offsets rise, the first is found by halving.
struct Pairs {
  const Table* tab;                      // NULL: more runs than it holds
  bool falls;
  int b, end, id, lo, hi;
  __device__ __forceinline__ int first_of(const FwdArgs& g, int i) const { return tab ? tab->begin[i] : g.low_runs.begin(i); }
  __device__ __forceinline__ int end_of(const FwdArgs& g, int i) const { return tab ? tab->end[i] : g.low_runs.end(i); }
  __device__ __forceinline__ int id_of(const FwdArgs& g, int i) const { return tab ? tab->cum[i] : g.low_ids[i]; }
  __device__ __forceinline__ Pairs(const FwdArgs& g, const Table& t, int n0, int nt, bool fall) : tab(g.low_runs.runs <= kMaxRuns ? &t : nullptr), falls(fall), end(n0 + nt) {
    int a = 0, c = falls ? 0 : g.low_runs.runs;            // the first run that ends behind n0
    while (a < c) {
      const int mid = (a + c) >> 1;
      if (end_of(g, mid) > n0) c = mid; else a = mid + 1;
    }
    b = a;
  }
  __device__ __forceinline__ bool next(const FwdArgs& g, int n0) {
    for (; b < g.low_runs.runs; ++b) {
      lo = max(first_of(g, b), n0);
      if (lo >= end && !falls) return false;
      hi = min(end_of(g, b), end);
      id = id_of(g, b);
      if (lo >= hi || id < 0 || id >= g.n) continue;
      for (++b; b < g.low_runs.runs && hi < end && id_of(g, b) == id && first_of(g, b) == hi; ++b) hi = max(hi, min(end_of(g, b), end));
      return true;
    }
    return false;
  }
};
// The part of a tile that a pair's columns are in, in whole grains: a tile of its own; whether columns of other runs are there too.
template <bool PAIR>
__device__ __forceinline__ Tile part_of(const Tile& o, const Pairs& p, bool& shared) {
  Tile t = o;
  t.n0 = o.n0 + ((p.lo - o.n0) & ~(kGrain<PAIR> - 1));
  t.nt = product_columns<PAIR>(p.hi - t.n0);
  shared = p.lo > t.n0 || p.hi < min(t.n0 + t.nt, o.n0 + o.nt);
  return t;
}
// whether the pair is left to the epilogue (for the tile; PAIR: both CTAs' rows)
template <bool PAIR>
__device__ __forceinline__ bool odd_pair(const FwdArgs& g, int m0, int id) {
  const unsigned char* f = g.odd + (long long)(m0 >> 7) * g.n + id;
  return (f[0] | (PAIR && m0 + 128 < g.M ? f[g.n] : 0)) != 0;
}
// K blocks that a pair adds: rank up to 32: both terms of T in one; above: the blocks of one, then those of the other
__device__ __forceinline__ int low_blocks(int r) { return r <= 32 ? 1 : 2 * ((r + 63) / 64); }

// Looks for infinities and NaN in the matrices of pairs that runs name, 128 rows of one to a warp: warp `w` of `warps`.  Where there are as many runs as pairs, in
// all pairs (200000 single columns of 20000 pairs: whether an earlier run has the pair took 9 ms).
template <bool BF16>
__device__ __forceinline__ void look_for_odd(const FwdArgs& g, long long w, long long warps) {
  constexpr uint32_t kExponent = BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
  auto high = [](uint32_t v) { return ((v & kExponent) + kOne) & 0x80008000u; };           // an exponent of ones runs over into the sign's place
  const bool all = g.low_runs.runs >= g.n;
  const int lane = threadIdx.x & 31, count = all ? g.n : g.low_runs.runs, blocks = (g.look_m + 127) >> 7;
  const bool vec = ((reinterpret_cast<uintptr_t>(g.low_B) & 15) | ((g.low_ldb | g.low_strideB) & 7)) == 0;
  const int parts = (int)min((long long)blocks, max(1ll, warps / max(1, count)));          // warps to a pair
  for (long long u = w; u < (long long)count * parts; u += warps) {
    const int part = parts > 1 ? (int)u / count : 0, b = (int)(u - (long long)part * count), id = all ? b : g.low_ids[b];
    if (id < 0 || id >= g.n) continue;
    bool again = false;                                    // an earlier run has the pair
    for (int i = 0; i < b && !all && !again; i += 32) again = __any_sync(0xffffffffu, i + lane < b && g.low_ids[i + lane] == id);
    if (again) continue;
    for (int rb = part; rb < blocks; rb += parts) {
      const int rows = min(128, g.look_m - rb * 128), inner = g.low_kmaj ? g.look_r : rows, outer = g.low_kmaj ? rows : g.look_r;
      const unsigned short* p = reinterpret_cast<const unsigned short*>(g.low_B) + id * g.low_strideB + rb * 128ll * (g.low_kmaj ? g.low_ldb : 1);
      const int pieces = vec ? inner >> 3 : 0;             // at most 16: 2^wide lanes to a line
      const int wide = pieces > 8 ? 4 : pieces > 4 ? 3 : pieces > 2 ? 2 : pieces > 1 ? 1 : 0, c = lane & ((1 << wide) - 1);
      uint32_t found = 0u;
      if (c < pieces) {
        const unsigned short* q = p + c * 8;
#pragma unroll 8
        for (int i = lane >> wide; i < outer; i += 32 >> wide) {
          const uint4 v = *reinterpret_cast<const uint4*>(q + i * g.low_ldb);
          found |= high(v.x) | high(v.y) | high(v.z) | high(v.w);
        }
      }
      if (inner > pieces * 8) {
#pragma unroll 4
        for (int i = 0; i < outer; ++i)
          for (int e = pieces * 8 + lane; e < inner; e += 32) found |= high(p[i * g.low_ldb + e]);
      }
      const int any = __any_sync(0xffffffffu, found != 0u);
      if (lane == 0) g.odd[(long long)rb * g.n + id] = any ? 1 : 0;
    }
  }
}
// Adds to a tile of products, in tensor memory, what the pairs that the tensor cores left out give: this warp's rows, every other 32 columns.  Hardly
// ever called.
template <bool BF16, bool PAIR>
__device__ __noinline__ void add_odd(const FwdArgs& g, const Table& tab, bool falls, int n0, int nt, int m0, int m, int part, uint32_t taddr) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  Pairs p(g, tab, n0, nt, falls);
  while (p.next(g, n0)) {
    if (!odd_pair<PAIR>(g, m0, p.id)) continue;
    const T* b = reinterpret_cast<const T*>(g.low_B) + (long long)p.id * g.low_strideB + (g.low_kmaj ? (long long)m * g.low_ldb : m);
    const long long step = g.low_kmaj ? 1 : g.low_ldb;
    for (int n = p.lo; n < p.hi; ++n) {
      const int c = n - n0;
      if (((c >> 5) & 1) != part) continue;
      const T* t = reinterpret_cast<const T*>(g.low_T) + (long long)n * g.low_width;
      float v = 0.f;
      if (m < g.M) {
#pragma unroll 4
        for (int k = 0; k < g.r; ++k) v = fmaf(Elem<T>::to_f(b[k * step]), Elem<T>::to_f(t[k]) + Elem<T>::to_f(t[g.low_step + k]), v);
      }
      __syncwarp();
      uint32_t a;
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(a) : "r"(taddr + c) : "memory");
      tmem_wait_ld();
      asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr + c), "r"(__float_as_uint(__uint_as_float(a) + v)) : "memory");
      tmem_wait_st();
    }
  }
}

// 16 lanes x 32 columns of tensor memory in the fragment layout of a matrix product: register 4 j + 2 s + e of lane l is row 8 s + l / 4,
// column 8 j + 2 (l % 4) + e
__device__ __forceinline__ void tmem_ld_frag32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// four 8 x 8 matrices to shared memory, transposed: lane 8 m + i gives the place of column i of matrix m
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t saddr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(saddr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}

// 32 rows x 32 columns of results of a warp of the epilogue to a column-major array.  The accumulator comes out of tensor memory in the
// fragment layout, which stmatrix transposes into a box of shared memory (a column's 32 rows are 64 bytes, whose 16-byte pieces trade
// places by column so that eight columns meet all banks); from there a warp stores eight columns of 64 bytes at a time.  f[0]: rows 0 .. 15,
// f[1]: 16 .. 31 of m..; columns n.., of which `wide` are written; bits of `gone`: zeros; vec: 16-byte stores are possible.
// (256 x 256: with stores of two rows, halves exchanged by shuffles, 8000 cycles; with boxes of 1 KB sent off by the copy engine 11500, for a
// fence and a copy each.)
template <bool BF16>
__device__ __forceinline__ void put_fragments(uint32_t (&f)[2][16], uint8_t* box, void* base, long long ld, int m, int n, int rows, int wide, uint32_t gone, bool vec) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const int lane = threadIdx.x & 31;
  if (m >= rows) return;
  if (gone) {
    const uint32_t bits = gone >> (2 * (lane & 3));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((bits >> (8 * (i >> 2) + (i & 1))) & 1u) f[h][i] = 0u;
  }
  // a lane's place in the first box half: matrices are rows 0 .. 7 and 8 .. 15 of columns 0 .. 7, then of 8 .. 15
  const int col = (lane & 7) + ((lane >> 4) << 3), piece = (lane >> 3) & 1, turn = (col >> 1) & 3;
  const uint32_t at = smem_u32(box) + col * 64;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = 4 * (2 * q + (x >> 1)) + 2 * (x & 1);
        v[x] = pack2<BF16>(__uint_as_float(f[h][i]), __uint_as_float(f[h][i + 1]));
      }
      stmatrix_x4_trans(at + q * 1024 + (((2 * h + piece) ^ turn) << 4), v[0], v[1], v[2], v[3]);
    }
  }
  __syncwarp();
  const int c = lane >> 2, r = (lane & 3) * 8;
  T* out = reinterpret_cast<T*>(base) + (long long)(n + c) * ld + m + r;
  const uint8_t* from = box + c * 64 + (((lane & 3) ^ ((c >> 1) & 3)) << 4);
  const bool whole = vec && m + r + 8 <= rows;
#pragma unroll
  for (int i = 0; i < 4; ++i, out += 8 * ld) {
    if (i * 8 + c >= wide) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(from + i * 512);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (whole) {
      *reinterpret_cast<uint4*>(out) = v;
    } else if (m + r + 8 <= rows) {
      // columns that begin at no multiple of 16 bytes: words, where a column of odd length begins between two of them put together anew
      // (dA of 10 matrices of 12343 x 2728: 1623 us element by element, 528 so)
      if (reinterpret_cast<uintptr_t>(out) & 2) {
        reinterpret_cast<unsigned short*>(out)[0] = (unsigned short)w[0];
#pragma unroll
        for (int e = 0; e < 3; ++e) *reinterpret_cast<uint32_t*>(reinterpret_cast<unsigned short*>(out) + 1 + 2 * e) = __funnelshift_r(w[e], w[e + 1], 16);
        reinterpret_cast<unsigned short*>(out)[7] = (unsigned short)(w[3] >> 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) reinterpret_cast<uint32_t*>(out)[e] = w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (m + r + e < rows) reinterpret_cast<unsigned short*>(out)[e] = (unsigned short)(w[e >> 1] >> (e & 1 ? 16 : 0));
    }
  }
  __syncwarp();
}
// Chunks of 32 columns through put(values, chunk), like drain_columns, in that layout
template <bool PAIR, typename F>
__device__ __forceinline__ void drain_fragments(uint32_t taddr, int c, int chunks, uint64_t* empty, F put) {
  constexpr int STEP = 2;
  uint32_t a[2][16], b[2][16];
  auto load = [&](uint32_t (&r)[2][16], int i) {
    tmem_ld_frag32(taddr + i * 32, r[0]);
    tmem_ld_frag32(taddr + (16u << 16) + i * 32, r[1]);
  };
  auto free = [&] {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      if (PAIR) arrive_first(empty);
      else mbar_arrive(empty);
    }
  };
  if (c >= chunks) {
    free();
    return;
  }
  load(a, c);
  while (true) {
    tmem_wait_ld();
    if (c + STEP < chunks) load(b, c + STEP); else free();
    put(a, c);
    if ((c += STEP) >= chunks) break;
    tmem_wait_ld();
    if (c + STEP < chunks) load(a, c + STEP); else free();
    put(b, c);
    if ((c += STEP) >= chunks) break;
  }
}

// Chunks c, c + 2, ... of 32 columns of this warp's rows of an accumulator through put(values, chunk): the next chunk is on
// its way out of tensor memory while one is put.  Then the accumulator is free as far as this warp goes.
template <bool PAIR, typename F>
__device__ __forceinline__ void drain_columns(uint32_t taddr, int c, int chunks, uint64_t* empty, F put) {
  constexpr int STEP = 2;
  uint32_t a[32], b[32];
  auto free = [&] {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      if (PAIR) arrive_first(empty);
      else mbar_arrive(empty);
    }
  };
  if (c >= chunks) {
    free();
    return;
  }
  tmem_ld32(taddr + c * 32, a);
  while (true) {
    tmem_wait_ld();
    if (c + STEP < chunks) tmem_ld32(taddr + (c + STEP) * 32, b); else free();
    put(a, c);
    if ((c += STEP) >= chunks) break;
    tmem_wait_ld();
    if (c + STEP < chunks) tmem_ld32(taddr + (c + STEP) * 32, a); else free();
    put(b, c);
    if ((c += STEP) >= chunks) break;
  }
}

template <bool BF16, int NT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
grouped_umma_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_t, const __grid_constant__ FwdArgs g) {
  using C = Cfg<NT, PAIR>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Table& tab = *reinterpret_cast<Table*>(smem + C::kTableOff);
  Bars* bars = reinterpret_cast<Bars*>(smem + C::kBarOff);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = (g.K + kBK - 1) / kBK;

  const int rank = PAIR ? cluster_rank() : 0, worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  let_next();
  set_up<NT, PAIR>(bars);
  const bool falls = count_tiles(g, tab, bars->search);
  if (g.wait == kWaitData) wait_before();
  tc_fence_before();
  sync_all<PAIR>();
  tc_fence_after();
  const uint32_t tmem = __reduce_or_sync(0xffffffffu, bars->tmem_base);     // (in a uniform register)
  const bool start_ok = (*abort_flag == 0);
  const long long columns = g.runs.offsets ? tab.cum[g.G] : (long long)g.G * tile_count((int)g.runs.len, g.cap);
  const long long tiles = columns * g.tiles_m * g.splits;

  if (start_ok && (warp == 0 || warp >= 10)) {
    // ----------------------------------------------------------- TMA producers
    const int me = warp == 0 ? 0 : warp - 9;
    if (lane == 0) {
      prefetch_tensormap(&tm_a);
      prefetch_tensormap(&tm_x);
    }
    bool ok = true;
    Ring<C::kStages> at;
    int turn = 0;
    // One stage, if it is this warp's turn: the boxes of the matrix (map ma, block ka of matrix za) and of the columns (map mx, block kx).  Lane 0 issues them all;
    // gathered columns are the other lanes' too, four each.
    auto fill = [&](const CUtensorMap* ma, int ka, int za, bool kmaj, const CUtensorMap* mx, int kx, const Tile& o, bool gather, const int4& four, bool side, int subs) {
      const bool mine = turn == me;
      if (++turn == kProducers) turn = 0;
      if (!mine) {
        at.next();
        return true;
      }
      const int s = at.s;
      uint8_t* da = smem + s * C::kStage;
      uint8_t* dx = da + C::kXOff;
      int good = 1;
      if (lane == 0) {
        if (at.round > 0) good = mbar_wait(&bars->empty[s], (uint32_t)(at.round - 1) & 1u, abort_flag) ? 1 : 0;
        if (good) {
          // (rows of shared memory behind the last row of the matrix keep what they have: no row sees another)
          const int mine = PAIR ? product_columns<true>(o.nt) / 2 : o.nt, n0 = o.n0 + rank * mine, m0 = o.m0 + rank * 128;
          const int boxes = (mine + C::kBox - 1) / C::kBox;
          auto of_a = [&](int first) {
            const int rows = max(0, min(128, g.M - first));
            return kmaj ? (rows + 127) / 128 : (rows + 63) / 64;
          };
          const int n_a = of_a(m0), box_a = kmaj ? kHalfBytes : kHalfBytes / 2;
          const int bytes = n_a * box_a + (gather ? round16(o.nt) * 128 : boxes * C::kBox * 128);
          if (!PAIR || side) {
            uint64_t* bar = PAIR && rank ? &bars->side[s] : &bars->full[s];
            mbar_arrive_expect_tx(bar, bytes);             // (one block: such stages of a pair are low-rank pairs')
            for (int i = 0; i < n_a; ++i) tma_load_3d(da + i * box_a, ma, bar, kmaj ? ka : m0 + i * 64, kmaj ? m0 : ka, za);
            if (!gather)
              for (int i = 0; i < boxes; ++i) tma_load_2d(dx + i * C::kBox * 128, mx, bar, kx, n0 + i * C::kBox);
          } else {
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], subs * (bytes + of_a(m0 + 128) * box_a + boxes * C::kBox * 128));
            const uint32_t bar = first_barrier(&bars->full[s]);
            for (int u = 0; u < subs; ++u, ka += kBK, kx += kBK) {
              for (int i = 0; i < n_a; ++i) pair_load_3d(da + u * C::kA + i * box_a, ma, bar, kmaj ? ka : m0 + i * 64, kmaj ? m0 : ka, za);
              for (int i = 0; i < boxes; ++i) pair_load_2d(dx + u * C::kX + i * C::kBox * 128, mx, bar, kx, n0 + i * C::kBox);
            }
          }
        }
      }
      at.next();
      if (gather) {
        good = __shfl_sync(0xffffffffu, good, 0);
        if (good && lane * 4 < round16(o.nt)) tma_gather4(dx + lane * 512, mx, &bars->full[s], kx, four);
      }
      return good != 0;
    };
    // (all lanes stay together where columns are gathered; elsewhere the others have nothing to do)
    if (g.gather || lane == 0) {
      for (long long t = worker; t < tiles && ok; t += workers) {
        const Tile o = tile_of<PAIR>(g, tab, t, nkb);
        if (o.nt <= 0) continue;
        int4 four = make_int4(0, 0, 0, 0);
        if (g.gather) {
          int c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = lane * 4 + e;
            c[e] = n < o.nt ? g.columns[o.n0 + n] : 0;
            if ((unsigned)c[e] >= (unsigned)g.N) c[e] = 0;     // (its column of C becomes zeros)
          }
          four = make_int4(c[0], c[1], c[2], c[3]);
        }
        for (int kb = o.kb0; kb < o.kb1 && ok; kb += C::kSub)
          ok = fill(&tm_a, kb * kBK, g.a_same ? 0 : o.mat, g.a_kmaj != 0, &tm_x, kb * kBK, o, g.gather != 0, four, false, min(C::kSub, o.kb1 - kb));
        if (g.r > 0 && ok) {
          Pairs p(g, tab, o.n0, o.nt, falls);
          const int blocks = low_blocks(g.r), half = blocks / 2;
          while (ok && p.next(g, o.n0)) {
            if (odd_pair<PAIR>(g, o.m0, p.id)) continue;
            bool shared;
            const Tile own = part_of<PAIR>(o, p, shared);
            for (int q = 0; q < blocks && ok; ++q) ok = fill(&tm_b, (half ? q % half : 0) * kBK, g.low_same ? 0 : p.id, g.low_kmaj != 0, &tm_t, q * kBK, own, false, four, shared, 1);
          }
        }
      }
    }
    __syncwarp();
    if (warp == 0 && lane == 0 && *abort_flag) {
      // give copies still in flight a bounded chance to land before the CTA leaves
      for (int i = 0; i < C::kStages; ++i) {
        const int rounds = at.round - (i < at.s ? 0 : 1);
        if (rounds >= 0) mbar_wait_drain(&bars->full[i], (uint32_t)rounds & 1u, kDrainNs);
      }
    }
  } else if (start_ok && warp == 1) {
    // -------------------------------------------------------------- MMA issuer; in the second CTA of a pair what clears its columns of a stage and says so
    bool ok = true;
    Ring<C::kStages> at;
    int ti = 0;
    const uint32_t base = desc_lo(smem_u32(smem));
    const bool issues = !PAIR || rank == 0;
    uint32_t sides = 0u;                                   // phases of the barriers `side`
    for (long long t = worker; t < tiles && ok; t += workers) {
      const Tile o = tile_of<PAIR>(g, tab, t, nkb);
      if (o.nt <= 0) continue;
      const int ab = ti & 1, wide = product_columns<PAIR>(o.nt);
      const uint32_t acc = tmem + ab * NT;
      if (issues) {
        const uint32_t id_main = idesc_of<PAIR>(BF16, wide, !g.a_kmaj, false);
        if (ti >= 2) ok = wait_of<PAIR>(&bars->acc_empty[ab], (uint32_t)((ti >> 1) + 1) & 1u, abort_flag);
        tc_fence_after();
        const uint32_t step = g.a_kmaj ? 32 >> 4 : 2048 >> 4;
        for (int kb = o.kb0; kb < o.kb1 && ok; kb += C::kSub) {
          const int s = at.s;
          ok = warp_wait(&bars->full[s], (uint32_t)at.round & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = base + s * (C::kStage >> 4), x = a + (C::kXOff >> 4);
          const int steps = (min(g.K, o.kb1 * kBK) - kb * kBK + 15) >> 4;    // of 16, four to a block
#pragma unroll
          for (int kk = 0; kk < 4 * C::kSub; ++kk)
            if (kk < steps)
              multiply_add<PAIR>(acc, a + (kk >> 2) * (C::kA >> 4) + (kk & 3) * step, x + (kk >> 2) * (C::kX >> 4) + (kk & 3) * 2, id_main, (kb > o.kb0 || kk > 0) ? 1u : 0u);
          commit_to<PAIR>(&bars->empty[s]);
          at.next();
        }
      } else {
        at.skip((o.kb1 - o.kb0 + C::kSub - 1) / C::kSub);
      }
      if (g.r > 0 && ok) {
        Pairs p(g, tab, o.n0, o.nt, falls);
        const int blocks = low_blocks(g.r), half = blocks / 2;
        const uint32_t step = g.low_kmaj ? 32 >> 4 : 2048 >> 4;
        while (ok && p.next(g, o.n0)) {
          if (odd_pair<PAIR>(g, o.m0, p.id)) {
            if (lane == 0) *reinterpret_cast<volatile int*>(&bars->odd) = 1;
            continue;
          }
          bool side;                                       // columns of other runs take no part
          const Tile own = part_of<PAIR>(o, p, side);
          const int mine = PAIR ? own.nt / 2 : own.nt, n0 = own.n0 + rank * mine, lo = p.lo - n0, hi = p.hi - n0;
          const uint32_t id_low = idesc_of<PAIR>(BF16, own.nt, !g.low_kmaj, false), d = acc + (own.n0 - o.n0);
          for (int q = 0; q < blocks; ++q, at.next()) {
            const int s = at.s;
            uint8_t* tx = smem + s * C::kStage + C::kXOff;
            if (!issues && !side) continue;
            ok = issues ? warp_wait(&bars->full[s], (uint32_t)at.round & 1u, abort_flag) : warp_wait(&bars->side[s], (sides >> s) & 1u, abort_flag);
            if (!ok) break;
            if (side) {
              for (int i = lane; i < mine * 8; i += 32)
                if ((i >> 3) < lo || (i >> 3) >= hi) *reinterpret_cast<uint4*>(tx + i * 16) = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
              __syncwarp();
              if (PAIR && !issues && lane == 0) arrive_first(&bars->side[s]);
              if (PAIR && issues) ok = wait_of<PAIR>(&bars->side[s], (sides >> s) & 1u, abort_flag);
              sides ^= 1u << s;
              if (!ok) break;
            }
            if (issues) {
              tc_fence_after();
              const uint32_t a = base + s * (C::kStage >> 4), x = a + (C::kXOff >> 4);
              const int left = half ? g.r - (q % half) * kBK : g.r, steps = min(4, (left + 15) >> 4);
              for (int kk = 0; kk < steps; ++kk) {
                multiply_add<PAIR>(d, a + kk * step, x + kk * 2, id_low, 1u);
                if (!half) multiply_add<PAIR>(d, a + kk * step, x + kk * 2 + 4, id_low, 1u);
              }
              commit_to<PAIR>(&bars->empty[s]);
            }
          }
        }
      }
      if (ok && issues) commit_to<PAIR>(&bars->acc_full[ab]);
      ++ti;
    }
  } else if (start_ok && warp >= 2 && warp < 10) {
    // ----------------------------------------------------------------- epilogue
    const int wq = warp & 3, part = (warp - 2) >> 2;       // TMEM lane quarter; every other 32 columns
    bool ok = true;
    int ti = 0;
    uint8_t* box = smem + C::kOutOff + (warp - 2) * 2048;
    if (g.look_r > 0) look_for_odd<BF16>(g, (gridDim.x - 1 - blockIdx.x) * 8ll + warp - 2, gridDim.x * 8ll);      // (the last CTAs have the fewest tiles)
    for (long long t = worker; t < tiles && ok; t += workers) {
      const Tile o = tile_of<PAIR>(g, tab, t, nkb);
      if (o.nt <= 0) continue;
      const int ab = ti & 1;
      uint32_t none[NT / 32];                              // columns whose column of X does not exist, a bit each
#pragma unroll
      for (int c = 0; c < NT / 32; ++c) {
        none[c] = 0u;
        if (g.columns && c * 32 < o.nt)
          none[c] = __ballot_sync(0xffffffffu, c * 32 + lane < o.nt && (unsigned)g.columns[o.n0 + min(c * 32 + lane, o.nt - 1)] >= (unsigned)g.N);
      }
      ok = mbar_wait_warp(&bars->acc_full[ab], (uint32_t)(ti >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const int m = o.m0 + rank * 128 + wq * 32 + lane;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(wq * 32) << 16) + ab * NT;
      const int chunks = m - lane < g.M ? (o.nt + 31) / 32 : 0;
      float scale = 1.f;
      if (g.to != kToC) scale = g.scale ? g.scale[o.mat] : g.scale0;
      if (g.to == kToC) {
        if (g.r > 0 && chunks > 0 && *reinterpret_cast<volatile int*>(&bars->odd)) add_odd<BF16, PAIR>(g, tab, falls, o.n0, o.nt, o.m0, m, part, taddr);
        auto put = [&](uint32_t (&f)[2][16], int c) {
          uint32_t gone = 0u;
#pragma unroll
          for (int q = 0; q < NT / 32; ++q)
            if (q == c) gone = none[q];
          put_fragments<BF16>(f, box, g.C, g.ldc, m - lane, o.n0 + c * 32, g.M, o.nt - c * 32, gone, g.vec != 0);
        };
        drain_fragments<PAIR>(taddr, part, chunks, &bars->acc_empty[ab], put);
        ++ti;
        continue;
      }
      auto put = [&](const uint32_t (&acc)[32], int c) {
        const int nc = min(32, o.nt - c * 32), n = o.n0 + c * 32;
        if (g.to == kToParts) {
          float* out = reinterpret_cast<float*>(g.C) + ((long long)o.split * g.runs.R + n) * g.M + m;
          if (m < g.M) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < nc) out[(long long)j * g.M] = scale * __uint_as_float(acc[j]);
          }
        } else if (m < g.low_step) {
          // T; zeros behind the rank
          T* out = reinterpret_cast<T*>(g.C) + (long long)n * g.low_width + m;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (j < nc) put_terms(out + (long long)j * g.low_width, g.low_step, m < g.M ? scale * __uint_as_float(acc[j]) : 0.f);
          }
        }
      };
      drain_columns<PAIR>(taddr, part, chunks, &bars->acc_empty[ab], put);
      ++ti;
    }
    if (g.zero_rest && ok) {
      // columns in no run: those before the first and behind the last one, or, where offsets fall, what a look at all of them says
      const int first = falls ? g.runs.R : tab.begin[0], last = falls ? g.runs.R : g.runs.at(g.G);
      const int rest = first + g.runs.R - last;
      for (int i = blockIdx.x * 8 + warp - 2; i < rest; i += gridDim.x * 8) {
        bool in = false;
        if (falls)
          for (int b = 0; b < g.G && !in; b += 32) in = __any_sync(0xffffffffu, b + lane < g.G && tab.begin[b + lane] <= i && i < tab.end[b + lane]);
        if (in) continue;
        T* out = reinterpret_cast<T*>(g.C) + (long long)(i < first ? i : last + i - first) * g.ldc;
        for (int m = lane; m < g.M; m += 32) out[m] = Elem<T>::from_f(0.f);
      }
    }
  }

  if (g.wait == kWaitEnd) wait_before();
  tear_down<NT, PAIR>(bars, tmem, g.status);
}

// ------------------------------------------------------------------------------------------------- gradient
//     A_a[row, col] = sum over the columns i of the runs of matrix a of P[row, i] Q[col, i]
// rows and columns of the matrix being features of dC and X, or of X and dC: the one that is stored contiguously is the rows'.  Both
// operands are MN-major, the contraction runs over a run's columns in blocks of 64; what a block holds behind the run's end is
// cleared in shared memory before it is multiplied (another run's infinity times zero would be a NaN).
struct GradArgs {
  Runs runs;
  const int* ids;
  void* A;
  long long ld, stride;                  // between columns and matrices of the result
  int rows, cols, G, mats;
  int tiles_r, tiles_c, vec;
  int wait;                              // launched early
  int fold, fold_at, fold_step, along;   // fold: columns fold_step apart, from fold_at on, are the two terms of one; along: a row's columns are contiguous
  float fold_scale;                      // of the second of them
  float* parts;                          // fold, in parts of the columns: (rows, cols, mats, splits) instead of A
  int splits;
  int* status;
};

template <bool BF16, int NT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
grouped_grad_umma_kernel(const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ GradArgs g) {
  using C = Cfg<NT, PAIR>;
  constexpr int kBlock = kBK * C::kSub;                    // columns of a stage
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Bars* bars = reinterpret_cast<Bars*>(smem + C::kBarOff);
  Table& tab = *reinterpret_cast<Table*>(smem + C::kTableOff);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? cluster_rank() : 0, worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  let_next();
  set_up<NT, PAIR>(bars);
  if (g.wait) wait_before();
  const bool held = g.G <= kMaxRuns;
  if (held) {
    for (int i = threadIdx.x; i < g.G; i += kThreads) {
      tab.cum[i] = g.ids ? g.ids[i] : i;
      tab.begin[i] = g.runs.begin(i);
      tab.end[i] = g.runs.end(i);
    }
  }
  tc_fence_before();
  sync_all<PAIR>();
  tc_fence_after();
  const uint32_t tmem = __reduce_or_sync(0xffffffffu, bars->tmem_base);     // (in a uniform register)
  const bool start_ok = (*abort_flag == 0);
  const long long each = (long long)g.tiles_r * g.tiles_c * g.splits, tiles = each * g.mats;
  auto begin_of = [&](int b) { return held ? tab.begin[b] : g.runs.begin(b); };
  auto end_of = [&](int b) { return held ? tab.end[b] : g.runs.end(b); };
  // The runs of matrix a that have columns, one after the other, -1: no more.  A warp looks at 32 at a time (64 runs of 64 pairs, 4096 x 16: one
  // at a time each tile took 17000 cycles to find its own, 121 us for what takes 35 so).
  struct Walk {
    int at = -32;
    unsigned found = 0u;
    int pos = 0, lo = 0, hi = 0x7fffffff;                  // blocks of columns gone by, and those that are wanted
  };
  auto next_run = [&](Walk& w, int a) {
    if (!g.ids) {
      const bool first = w.at < 0;
      w.at = 0;
      return first && a < g.G && end_of(a) > begin_of(a) ? a : -1;
    }
    while (w.found == 0u) {
      if ((w.at += 32) >= g.G) return -1;
      const int b = w.at + lane;
      w.found = __ballot_sync(0xffffffffu, b < g.G && (held ? tab.cum[b] : g.ids[b]) == a && end_of(b) > begin_of(b));
    }
    const int b = w.at + __ffs(w.found) - 1;
    w.found &= w.found - 1u;
    return b;
  };
  // part `split` of the blocks of matrix a
  auto walk_of = [&](int a, int split) {
    Walk w;
    if (g.splits > 1) {
      Walk all;
      int n = 0;
      for (int b = next_run(all, a); b >= 0; b = next_run(all, a)) n += (end_of(b) - begin_of(b) + kBlock - 1) / kBlock;
      w.lo = (int)((long long)n * split / g.splits);
      w.hi = (int)((long long)n * (split + 1) / g.splits);
    }
    return w;
  };
  // the next columns of a run that are wanted: false: no more
  auto next_piece = [&](Walk& w, int a, int& begin, int& end) {
    while (w.pos < w.hi) {
      const int b = next_run(w, a);
      if (b < 0) return false;
      begin = begin_of(b);
      end = end_of(b);
      if (g.splits == 1) return true;
      const int n = (end - begin + kBlock - 1) / kBlock, first = max(0, w.lo - w.pos), last = min(n, w.hi - w.pos);
      w.pos += n;
      if (first >= last) continue;
      if (last < n) end = begin + last * kBlock;
      begin += first * kBlock;
      return true;
    }
    return false;
  };

  if (start_ok && (warp == 0 || warp >= 10)) {
    const int me = warp == 0 ? 0 : warp - 9;
    if (lane == 0) {
      prefetch_tensormap(&tm_r);
      prefetch_tensormap(&tm_c);
    }
    __syncwarp();
    bool ok = true;
    Ring<C::kStages> at;
    int turn = 0;
    for (long long t = worker; t < tiles && ok; t += workers) {
      const int a = (int)(t / each), in = (int)(t - a * each), q = g.splits > 1 ? in / g.splits : in, split = in - q * g.splits;
      const int r0 = (q % g.tiles_r) * (PAIR ? 256 : 128) + rank * 128, left = g.cols - (q / g.tiles_r) * NT;
      const int c0 = g.fold_at + (q / g.tiles_r) * NT + (PAIR ? rank * (product_columns<true>(min(NT, left)) / 2) : 0);
      Walk walk = walk_of(a, split);
      int begin, end;
      while (ok && next_piece(walk, a, begin, end)) {
        for (int i0 = begin; i0 < end; i0 += kBlock, at.next()) {
          const bool mine = turn == me;
          if (++turn == kProducers) turn = 0;
          if (!mine) continue;
          const int s = at.s;
          if (lane == 0) {
            if (at.round > 0) ok = mbar_wait(&bars->empty[s], (uint32_t)(at.round - 1) & 1u, abort_flag);
            if (ok) {
              uint8_t* d = smem + s * C::kStage;
              const bool side = ((end - i0) & 15) && end - i0 < kBlock;
              const int subs = min(C::kSub, (end - i0 + kBK - 1) / kBK);
              if (!PAIR || side) {
                uint64_t* bar = PAIR && rank ? &bars->side[s] : &bars->full[s];
                mbar_arrive_expect_tx(bar, subs * (C::kA + C::kX));
                for (int u = 0; u < subs; ++u) {
#pragma unroll
                  for (int x = 0; x < 2; ++x) tma_load_2d(d + u * C::kA + x * (kHalfBytes / 2), &tm_r, bar, r0 + x * 64, i0 + u * kBK);
#pragma unroll
                  for (int x = 0; x < C::kX / (kHalfBytes / 2); ++x) tma_load_2d(d + C::kXOff + u * C::kX + x * (kHalfBytes / 2), &tm_c, bar, c0 + x * 64, i0 + u * kBK);
                }
              } else {
                if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * subs * (C::kA + C::kX));
                const uint32_t bar = first_barrier(&bars->full[s]);
                for (int u = 0; u < subs; ++u) {
#pragma unroll
                  for (int x = 0; x < 2; ++x) pair_load_2d(d + u * C::kA + x * (kHalfBytes / 2), &tm_r, bar, r0 + x * 64, i0 + u * kBK);
#pragma unroll
                  for (int x = 0; x < C::kX / (kHalfBytes / 2); ++x) pair_load_2d(d + C::kXOff + u * C::kX + x * (kHalfBytes / 2), &tm_c, bar, c0 + x * 64, i0 + u * kBK);
                }
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
          if (!ok) break;
        }
      }
    }
    if (me == 0 && lane == 0 && *abort_flag) {
      for (int i = 0; i < C::kStages; ++i) {
        const int rounds = at.round - (i < at.s ? 0 : 1);
        if (rounds >= 0) mbar_wait_drain(&bars->full[i], (uint32_t)rounds & 1u, kDrainNs);
      }
    }
  } else if (start_ok && warp == 1) {
    bool ok = true;
    Ring<C::kStages> at;
    int ti = 0;
    const uint32_t base = desc_lo(smem_u32(smem));
    const bool issues = !PAIR || rank == 0;
    uint32_t sides = 0u;                                   // phases of the barriers `side`
    for (long long t = worker; t < tiles && ok; t += workers, ++ti) {
      const int a = (int)(t / each), in = (int)(t - a * each), q = g.splits > 1 ? in / g.splits : in, split = in - q * g.splits, left = g.cols - q / g.tiles_r * NT;
      const int ab = ti & 1;
      const uint32_t acc = tmem + ab * NT;
      const uint32_t idesc = idesc_of<PAIR>(BF16, g.fold ? NT : product_columns<PAIR>(min(NT, left)), true, true);
      if (ti >= 2 && issues) ok = wait_of<PAIR>(&bars->acc_empty[ab], (uint32_t)((ti >> 1) + 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      bool begun = false;
      Walk walk = walk_of(a, split);
      int begin, end;
      while (ok && next_piece(walk, a, begin, end)) {
        // a block of which the first `here` columns are the run's
        auto multiply = [&](int here) {
          tc_fence_after();
          const uint32_t r = base + at.s * (C::kStage >> 4), c = r + (C::kXOff >> 4);
#pragma unroll
          for (int kk = 0; kk < 4 * C::kSub; ++kk)
            if (kk * 16 < here)
              multiply_add<PAIR>(acc, r + (kk >> 2) * (C::kA >> 4) + (kk & 3) * (2048 >> 4), c + (kk >> 2) * (C::kX >> 4) + (kk & 3) * (2048 >> 4), idesc, (begun || kk > 0) ? 1u : 0u);
          commit_to<PAIR>(&bars->empty[at.s]);
          begun = true;
        };
        const int whole = (end - begin) / kBlock, rest = (end - begin) % kBlock;
        if (issues) {
          for (int i = 0; i < whole && ok; ++i) {
            ok = warp_wait(&bars->full[at.s], (uint32_t)at.round & 1u, abort_flag);
            if (!ok) break;
            multiply(kBlock);
            at.next();
          }
        } else {
          at.skip(whole);
        }
        const bool side = rest & 15;                       // behind the run's end: another run's columns, or nobody's
        if (ok && rest && (issues || side)) {
          ok = issues ? warp_wait(&bars->full[at.s], (uint32_t)at.round & 1u, abort_flag) : warp_wait(&bars->side[at.s], (sides >> at.s) & 1u, abort_flag);
          if (!ok) break;
          if (side) {
            const int u = rest / kBK, there = rest % kBK;  // (a part of 16: in one block)
            for (int i = there * 8 + lane; i < round16(there) * 8; i += 32) {
#pragma unroll
              for (int x = 0; x < 2; ++x) *reinterpret_cast<uint4*>(smem + at.s * C::kStage + u * C::kA + x * (kHalfBytes / 2) + i * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll
              for (int x = 0; x < C::kX / (kHalfBytes / 2); ++x)
                *reinterpret_cast<uint4*>(smem + at.s * C::kStage + C::kXOff + u * C::kX + x * (kHalfBytes / 2) + i * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (PAIR && !issues && lane == 0) arrive_first(&bars->side[at.s]);
            if (PAIR && issues) ok = wait_of<PAIR>(&bars->side[at.s], (sides >> at.s) & 1u, abort_flag);
            sides ^= 1u << at.s;
            if (!ok) break;
          }
          if (issues) multiply(rest);
        }
        if (rest) at.next();
      }
      if (ok && issues) commit_to<PAIR>(&bars->acc_full[ab]);
    }
  } else if (start_ok && warp >= 2 && warp < 10) {
    const int wq = warp & 3, part = (warp - 2) >> 2;
    bool ok = true;
    int ti = 0;
    uint8_t* box = smem + C::kOutOff + (warp - 2) * 2048;
    for (long long t = worker; t < tiles && ok; t += workers, ++ti) {
      const int a = (int)(t / each), in = (int)(t - a * each), q = g.splits > 1 ? in / g.splits : in, split = in - q * g.splits;
      const int r0 = (q % g.tiles_r) * (PAIR ? 256 : 128) + rank * 128, c0 = (q / g.tiles_r) * NT;
      const int ab = ti & 1;
      Walk walk = walk_of(a, split);
      int begin, end;
      const bool some = next_piece(walk, a, begin, end);   // a matrix that no column met is zeros
      ok = mbar_wait_warp(&bars->acc_full[ab], (uint32_t)(ti >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const int m = r0 + wq * 32 + lane;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(wq * 32) << 16) + ab * NT;
      T* base = reinterpret_cast<T*>(g.A) + (long long)a * g.stride;
      const int width = g.fold ? g.fold_step : min(NT, g.cols - c0), chunks = m - lane < g.rows ? (width + 31) / 32 : 0;
      if (!g.fold) {
        auto put = [&](uint32_t (&f)[2][16], int c) {
          put_fragments<BF16>(f, box, base, g.ld, m - lane, c0 + c * 32, g.rows, g.cols - c0 - c * 32, some ? 0u : 0xffffffffu, g.vec != 0);
        };
        drain_fragments<PAIR>(taddr, part, chunks, &bars->acc_empty[ab], put);
        continue;
      }
      // (46 pairs of rank 128 and 5984 rows, stored along the rank: 468 us with stores of an element, 213 so)
      for (int c = part; c < chunks; c += 2) {
        const int n = c0 + c * 32;
        if (!g.along && !g.parts) {
          uint32_t f[2][16], more[2][16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            tmem_ld_frag32(taddr + (h << 20) + c * 32, f[h]);
            tmem_ld_frag32(taddr + (h << 20) + g.fold_step + c * 32, more[h]);
          }
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) f[h][i] = __float_as_uint(both_terms(f[h][i], more[h][i], g.fold_scale));
          put_fragments<BF16>(f, box, base, g.ld, m - lane, n, g.rows, g.cols - n, some ? 0u : 0xffffffffu, g.vec != 0);
          continue;
        }
        uint32_t acc[32], more[32];
        tmem_ld32(taddr + c * 32, acc);
        tmem_ld32(taddr + g.fold_step + c * 32, more);
        tmem_wait_ld();
        const int nc = min(32, g.cols - n);
        if (g.parts) {
          float* out = g.parts + (((long long)split * g.mats + a) * g.cols + n) * g.rows + m;
          if (m < g.rows) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < nc) out[(long long)j * g.rows] = some ? both_terms(acc[j], more[j], g.fold_scale) : 0.f;
          }
          __syncwarp();
          continue;
        }
        if (m < g.rows) {
          T* dst = base + (long long)m * g.ld + n;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = some ? both_terms(acc[j + e], more[j + e], g.fold_scale) : 0.f;
            if (g.vec && j + 8 <= nc) {
              *reinterpret_cast<uint4*>(dst + j) = make_uint4(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]), pack2<BF16>(v[4], v[5]), pack2<BF16>(v[6], v[7]));
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (j + e < nc) dst[j + e] = Elem<T>::from_f(v[e]);
            }
          }
        }
        __syncwarp();
      }
      __syncwarp();
      tc_fence_before();
      if (lane == 0) mbar_arrive(&bars->acc_empty[ab]);
    }
  }
  tear_down<NT, PAIR>(bars, tmem, g.status);
}

// The parts of such a gradient, added in their order.  A block takes 32 rows of a matrix and 32 columns at a time, turned in shared memory where a row's
// columns are contiguous.
struct JoinGradArgs {
  const float* parts;
  void* A;
  long long ld, stride;
  int rows, cols, mats, splits, along;
};
template <typename T>
__global__ void __launch_bounds__(256) join_grad_kernel(const __grid_constant__ JoinGradArgs g) {
  __shared__ float tile[32][33];
  let_next();
  wait_before();
  const int m0 = blockIdx.x * 32, a = blockIdx.y, x = threadIdx.x & 31, y = threadIdx.x >> 5;
  T* A = reinterpret_cast<T*>(g.A) + (long long)a * g.stride;
  for (int n0 = 0; n0 < g.cols; n0 += 32) {
    __syncthreads();
#pragma unroll
    for (int i = y; i < 32; i += 8) {
      float v = 0.f;
      if (n0 + i < g.cols && m0 + x < g.rows) {
#pragma unroll 4
        for (int s = 0; s < g.splits; ++s) v += g.parts[(((long long)s * g.mats + a) * g.cols + n0 + i) * g.rows + m0 + x];
        if (!g.along) A[(long long)(n0 + i) * g.ld + m0 + x] = Elem<T>::from_f(v);
      }
      if (g.along) tile[i][x] = v;
    }
    if (!g.along) continue;
    __syncthreads();
#pragma unroll
    for (int i = y; i < 32; i += 8)
      if (m0 + i < g.rows && n0 + x < g.cols) A[(long long)(m0 + i) * g.ld + n0 + x] = Elem<T>::from_f(tile[x][i]);
  }
}

// ------------------------------------------------------------------------------------------------- copies, host
// `count` matrices of wide x deep 16-bit elements to rows that the copy engine can address; with `of`, only those of runs that have
// columns; with `columns`, row i from row columns[i] of `rows`, zeros where there is none.
struct CopyArgs {
  const unsigned short* src;
  long long ld, stride, deep;
  uint4* dst;
  int wide, ld8, vec, rows;              // ld8: 16-byte packets of a row; vec: the source has them too
  const int* columns;
  Runs of;
};
// Rows at addresses that are no multiples of 16 bytes are read in words of four, 128 at a time by a warp, and put together by way of shared
// memory (3162 rows of 7046 elements: 39 us element by element, 28 so).
__global__ void __launch_bounds__(256) copy_rows_kernel(const __grid_constant__ CopyArgs g) {
  __shared__ __align__(16) uint32_t words[8][132];
  const int mat = blockIdx.z, lane = threadIdx.x & 31;
  uint32_t* mine = words[threadIdx.x >> 5];
  let_next();
  wait_before();
  if (g.of.offsets && g.of.end(mat) <= g.of.begin(mat)) return;
  const unsigned short* s = g.src + (long long)mat * g.stride;
  uint4* d = g.dst + (long long)mat * g.deep * g.ld8;
  for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < g.deep; row += (long long)gridDim.x * 8) {
    long long from = row;
    if (g.columns) {
      const int c = g.columns[row];
      from = (unsigned)c < (unsigned)g.rows ? c : -1;
    }
    const unsigned short* p = s + from * g.ld;
    uint4* to = d + row * g.ld8;
    if (g.vec || from < 0) {
      // four packets of a row at a time under way
#pragma unroll 4
      for (int i = lane; i < g.ld8; i += 32) to[i] = from >= 0 ? *reinterpret_cast<const uint4*>(p + i * 8) : make_uint4(0, 0, 0, 0);
      continue;
    }
    const int odd = (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 1;        // the first word begins an element before the row
    auto word = [&](int i) {
      const int e = 2 * i - odd;
      if (e >= 0 && e + 1 < g.wide) return *reinterpret_cast<const uint32_t*>(p + e);
      return (e >= 0 && e < g.wide ? (uint32_t)p[e] : 0u) | (e + 1 >= 0 && e + 1 < g.wide ? (uint32_t)p[e + 1] << 16 : 0u);
    };
    for (int i0 = 0; i0 < g.ld8; i0 += 32) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = word(i0 * 4 + u * 32 + lane);
      const uint32_t last = lane == 0 && odd ? word(i0 * 4 + 128) : 0u;
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 4; ++u) mine[u * 32 + lane] = w[u];
      if (lane == 0) mine[128] = last;
      __syncwarp();
      uint4 v = *reinterpret_cast<const uint4*>(&mine[lane * 4]);
      if (odd) {
        const uint32_t next = mine[lane * 4 + 4];
        v = make_uint4(__funnelshift_r(v.x, v.y, 16), __funnelshift_r(v.y, v.z, 16), __funnelshift_r(v.z, v.w, 16), __funnelshift_r(v.w, next, 16));
      }
      if (i0 + lane < g.ld8) to[i0 + lane] = v;
    }
  }
}

// Parts of a product whose K was cut, added in their order: C, and for columns of low-rank pairs B T on top (few columns: a pair's
// products are so little that they need no tensor cores).  A block takes a column and 256 rows.
struct JoinArgs {
  const float* parts;                    // (M, R, splits)
  void* C;
  long long ldc;
  int splits, M, R, N, zero_rest;
  Runs runs;
  const int* columns;
  const float* t;                        // (r, R, t_splits), r = 0: none
  int t_splits, r, n, transB;
  Runs low_runs;
  const int* low_ids;
  const void* B;
  long long ldb, strideB;
  int b_pairs, b_packets;                // rows of B come in pairs at an address of their size's multiple; transposed: 16 bytes along the rank do
};
template <typename T>
struct alignas(2 * sizeof(T)) Two {
  T x, y;
};
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ JoinArgs g) {
  __shared__ float t[128];
  __shared__ int pair;
  let_next();
  wait_before();
  const int n = blockIdx.x, m = (blockIdx.y * 128 + threadIdx.x) * 2;
  T* out = reinterpret_cast<T*>(g.C) + (long long)n * g.ldc + m;
  int in = 1;
  if (g.runs.offsets) {
    in = 0;
    for (int i = threadIdx.x; i < g.runs.runs; i += 128) in |= g.runs.begin(i) <= n && n < g.runs.end(i);
    in = __syncthreads_or(in);
    if (!in && !g.zero_rest) return;
  }
  if (g.r > 0) {
    if (g.low_runs.offsets) {
      if (threadIdx.x == 0) pair = -1;
      __syncthreads();
      for (int i = threadIdx.x; i < g.low_runs.runs; i += 128)
        if (g.low_runs.begin(i) <= n && n < g.low_runs.end(i)) pair = g.low_ids[i];
    } else if (threadIdx.x == 0) {
      const long long i = g.low_runs.len > 0 ? n / g.low_runs.len : g.low_runs.runs;
      pair = i < g.low_runs.runs ? g.low_ids[i] : -1;
    }
    if (threadIdx.x < g.r) {
      float v = 0.f;
#pragma unroll 4
      for (int s = 0; s < g.t_splits; ++s) v += g.t[((long long)s * g.R + n) * g.r + threadIdx.x];
      t[threadIdx.x] = v;
    }
    __syncthreads();
  }
  float sum[2] = {0.f, 0.f};
  if (in && (!g.columns || (unsigned)g.columns[n] < (unsigned)g.N)) {
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
      const float* p = g.parts + ((long long)s * g.R + n) * g.M + m;
      if (m < g.M) sum[0] += p[0];
      if (m + 1 < g.M) sum[1] += p[1];
    }
  }
  const int id = g.r > 0 ? pair : -1;
  if (id >= 0 && id < g.n && m < g.M) {
    const T* B = reinterpret_cast<const T*>(g.B) + (long long)id * g.strideB;
    const bool two = m + 1 < g.M;
    if (!g.transB && two && g.b_pairs) {
      const Two<T>* b = reinterpret_cast<const Two<T>*>(B + m);
#pragma unroll 8
      for (int i = 0; i < g.r; ++i) {
        const Two<T> v = b[i * (g.ldb / 2)];
        sum[0] = fmaf(Elem<T>::to_f(v.x), t[i], sum[0]);
        sum[1] = fmaf(Elem<T>::to_f(v.y), t[i], sum[1]);
      }
    } else if (g.transB && g.b_packets) {
      // (165 columns, 6384 x 64, Float32: 75 us, 251 element by element)
      constexpr int V = 16 / sizeof(T);
      const T* b = B + m * g.ldb;
#pragma unroll 4
      for (int i = 0; i < g.r; i += V) {
        const uint4 p = *reinterpret_cast<const uint4*>(b + i), q = two ? *reinterpret_cast<const uint4*>(b + g.ldb + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < V; ++u) {
          sum[0] = fmaf(Elem<T>::to_f(reinterpret_cast<const T*>(&p)[u]), t[i + u], sum[0]);
          sum[1] = fmaf(Elem<T>::to_f(reinterpret_cast<const T*>(&q)[u]), t[i + u], sum[1]);
        }
      }
    } else {
      const long long row = g.transB ? g.ldb : 1, col = g.transB ? 1 : g.ldb;
      const T* b = B + m * row;
#pragma unroll 8
      for (int i = 0; i < g.r; ++i) {
        sum[0] = fmaf(Elem<T>::to_f(b[i * col]), t[i], sum[0]);
        if (two) sum[1] = fmaf(Elem<T>::to_f(b[row + i * col]), t[i], sum[1]);
      }
    }
  }
  if (m < g.M) out[0] = Elem<T>::from_f(sum[0]);
  if (m + 1 < g.M) out[1] = Elem<T>::from_f(sum[1]);
}
// scale * A X of columns that hardly share a pair, in parts as the products leave them: a block takes a column and kLowK of K.  What bounds it is
// reading A, so it needs no tensor cores (64 requests of one column, rank 16, K = 4096: 20 us as a product, 8.6 so).
constexpr int kLowK = 1024;
struct LowFewArgs {
  const void* A;
  const void* X;
  float* parts;                          // (r, R, splits)
  long long lda, strideA, ldx;
  const float* scale;
  float scale0;
  Runs runs;
  const int* ids;
  int transA, r, K, R, mats, vec;        // vec: 16-byte packets of A along what is contiguous
};
template <typename T>
__global__ void __launch_bounds__(256) low_few_kernel(const __grid_constant__ LowFewArgs g) {
  __shared__ float x[kLowK];
  __shared__ float part[256 * 8], sums[256];
  __shared__ int pair;
  let_next();
  const int n = blockIdx.x, k0 = blockIdx.y * kLowK, nk = min(kLowK, g.K - k0), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    pair = -1;
    if (!g.runs.offsets) {
      const long long i = g.runs.len > 0 ? n / g.runs.len : g.runs.runs;
      if (i < g.runs.runs) pair = g.ids[i];
    }
  }
  __syncthreads();
  if (g.runs.offsets) {
    for (int i = threadIdx.x; i < g.runs.runs; i += 256)
      if (g.runs.begin(i) <= n && n < g.runs.end(i)) pair = g.ids[i];
  }
  const T* X = reinterpret_cast<const T*>(g.X) + (long long)n * g.ldx + k0;
  for (int k = threadIdx.x; k < nk; k += 256) x[k] = Elem<T>::to_f(X[k]);
  __syncthreads();
  const int id = pair;
  if (id < 0 || id >= g.mats) return;
  const float scale = g.scale ? g.scale[id] : g.scale0;
  const T* A = reinterpret_cast<const T*>(g.A) + (long long)id * g.strideA;
  float* out = g.parts + ((long long)blockIdx.y * g.R + n) * g.r;
  if (g.transA) {                        // K contiguous: a warp a row
    for (int i = warp; i < g.r; i += 8) {
      const T* a = A + (long long)i * g.lda + k0;
      float sum = 0.f;
      if (g.vec) {
#pragma unroll 4
        for (int k = lane * 8; k < nk; k += 256) {
          const uint4 v = *reinterpret_cast<const uint4*>(a + k);
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int u = 0; u < 8; ++u) sum = fmaf(Elem<T>::to_f(e[u]), x[k + u], sum);
        }
      } else {
#pragma unroll 4
        for (int k = lane; k < nk; k += 32) sum = fmaf(Elem<T>::to_f(a[k]), x[k], sum);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) out[i] = scale * sum;
    }
    return;
  }
  // the rank contiguous: eight (or one) of it to a thread, every L-th of K
  const int each = g.vec ? 8 : 1, groups = g.r / each, L = 256 / groups, group = threadIdx.x % groups, kl = threadIdx.x / groups;
  float acc[8] = {};
  if (kl < L) {
    const T* a = A + (long long)k0 * g.lda + group * each;
    if (g.vec) {
#pragma unroll 8
      for (int k = kl; k < nk; k += L) {
        const uint4 v = *reinterpret_cast<const uint4*>(a + (long long)k * g.lda);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int u = 0; u < 8; ++u) acc[u] = fmaf(Elem<T>::to_f(e[u]), x[k], acc[u]);
      }
    } else {
#pragma unroll 8
      for (int k = kl; k < nk; k += L) acc[0] = fmaf(Elem<T>::to_f(a[(long long)k * g.lda]), x[k], acc[0]);
    }
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) part[u * 256 + threadIdx.x] = acc[u];
  __syncthreads();
  // element i of the rank is component i % each of threads i / each + groups * (0 .. L - 1): cut into P, then P into one
  const int P = 256 / g.r, i = threadIdx.x % g.r, p = threadIdx.x / g.r;
  float sum = 0.f;
  if (p < P)
    for (int q = p; q < L; q += P) sum += part[(i % each) * 256 + i / each + groups * q];
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x < g.r) {
    sum = 0.f;
    for (int q = 0; q < P; ++q) sum += sums[q * g.r + threadIdx.x];
    out[threadIdx.x] = scale * sum;
  }
}
// T from the parts of scale * A X: two 16-bit terms, zeros behind the rank
template <typename T>
__global__ void __launch_bounds__(256) join_low_kernel(const float* parts, int splits, int r, int R, T* out, int width, int step) {
  let_next();
  wait_before();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int n = (int)(i / step), c = (int)(i % step);
  if (n >= R) return;
  float v = 0.f;
  if (c < r) {
#pragma unroll 4
    for (int s = 0; s < splits; ++s) v += parts[((long long)s * R + n) * r + c];
  }
  put_terms(out + (long long)n * width + c, step, v);
}

// A matrix (or several) that is read: where it lies, contiguous extent first.
struct Operand {
  const void* p;
  long long wide, deep, ld, stride, count;               // stride 0: all are one, which is copied once
  const int* columns;                    // rows `deep` of them are gathered from these of `rows`; NULL: as they lie
  long long rows;
  bool fits() const { return aligned16(p) && stride_ok(ld) && (count <= 1 || stride == 0 || stride_ok(stride)); }
  long long different() const { return stride ? count : std::min(count, 1ll); }
  size_t copy_bytes() const { return (fits() && !columns) || wide == 0 || deep == 0 || count == 0 ? 0 : (size_t)((wide + 7) / 8 * 16) * deep * different(); }
};
cudaError_t align_operand(Operand& o, char*& ws, const Runs* of, bool& behind, cudaStream_t st) {
  const size_t bytes = o.copy_bytes();
  if (!bytes) return cudaSuccess;
  CopyArgs c;
  c.src = static_cast<const unsigned short*>(o.p);
  c.ld = o.ld; c.stride = o.stride; c.deep = o.deep;
  c.dst = reinterpret_cast<uint4*>(ws);
  c.wide = (int)o.wide;
  c.ld8 = (int)((o.wide + 7) / 8);
  c.vec = o.fits() && o.wide % 8 == 0;
  c.rows = (int)o.rows;
  c.columns = o.columns;
  c.of = of && o.stride ? *of : Runs{nullptr, 0, 0, 0};
  const long long blocks = std::min<long long>((o.deep + 7) / 8, 1 << 20);
  // (behind: a kernel of this call is before it in the stream)
  const dim3 grid((unsigned)blocks, 1, (unsigned)o.different());
  if (behind) {
    const cudaError_t e = launch_early(copy_rows_kernel, grid, dim3(256), 0, st, c);
    if (e != cudaSuccess) return e;
  } else {
    copy_rows_kernel<<<grid, 256, 0, st>>>(c);
  }
  count_launch();
  behind = true;
  o.p = ws;
  o.ld = (long long)c.ld8 * 8;
  if (o.stride) o.stride = o.ld * o.deep;
  o.columns = nullptr;
  ws += (bytes + 255) / 256 * 256;
  return cudaGetLastError();
}
size_t padded(size_t n) { return (n + 255) / 256 * 256; }

bool encode(CUtensorMap* m, int dtype, int rank, const Operand& o, const cuuint32_t* box) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const long long stride = o.count > 1 && o.stride ? o.stride : o.ld * o.deep;
  const cuuint64_t dims[3] = {(cuuint64_t)o.wide, (cuuint64_t)o.deep, (cuuint64_t)(o.stride ? o.count : 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)stride * 2};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, dtype == NNLIB_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(o.p), dims, strides,
            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_matrix(CUtensorMap* m, int dtype, const Operand& o, bool kmaj) {
  const cuuint32_t box[3] = {64, kmaj ? 128u : 64u, 1};
  return encode(m, dtype, 3, o, box);
}
bool encode_columns(CUtensorMap* m, int dtype, const Operand& o, int rows) {
  const cuuint32_t box[2] = {64, (cuuint32_t)rows};
  return encode(m, dtype, 2, o, box);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
  return n;
}

struct Maps {
  CUtensorMap a, x, b, t;
};

template <bool PAIR, typename K, typename... Args>
cudaError_t launch(K kern, long long workers, int smem, bool early, cudaStream_t st, const Args&... args) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const long long most = sm_count() / (PAIR ? 2 : 1);
  const unsigned grid = (unsigned)std::max<long long>(1, std::min(workers, most)) * (PAIR ? 2 : 1);
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute a[2];
  c.attrs = a;
  if (PAIR) {
    a[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    a[c.numAttrs].val.clusterDim.x = 2;
    a[c.numAttrs].val.clusterDim.y = a[c.numAttrs].val.clusterDim.z = 1;
    ++c.numAttrs;
  }
  if (early) {
    a[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++c.numAttrs;
  }
  e = cudaLaunchKernelEx(&c, kern, args...);
  count_launch();
  return e == cudaSuccess ? cudaGetLastError() : e;
}
template <bool BF16, int NT, bool PAIR>
cudaError_t launch_fwd(const Maps& m, FwdArgs g, long long most, cudaStream_t st) {
  g.tiles_m = (g.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
  // (as many CTAs as look through the pairs' matrices in one go, be the tiles few)
  const long long looks = g.look_r > 0 ? ((long long)std::min(g.low_runs.runs, g.n) * ((g.look_m + 127) / 128) + 7) / 8 : 0;
  return launch<PAIR>(grouped_umma_kernel<BF16, NT, PAIR>, most * g.tiles_m * g.splits + looks, Cfg<NT, PAIR>::kSmem, g.wait != kWaitNone, st, m.a, m.x, m.b, m.t, g);
}
template <bool BF16, int NT, bool PAIR>
cudaError_t launch_bwd(const CUtensorMap& r, const CUtensorMap& c, GradArgs g, cudaStream_t st) {
  g.tiles_r = (g.rows + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
  g.tiles_c = g.fold ? 1 : (g.cols + NT - 1) / NT;
  return launch<PAIR>(grouped_grad_umma_kernel<BF16, NT, PAIR>, (long long)g.tiles_r * g.tiles_c * g.splits * g.mats, Cfg<NT, PAIR>::kSmem, g.wait != 0, st, r, c, g);
}

// Rows and columns of a tile.
struct Shape {
  bool pair;
  int cap, splits;
  long long most;                        // column tiles that there can be
  int nt() const { return cap > 128 ? 256 : cap > 64 ? 128 : cap > 32 ? 64 : 32; }
};
// The tile, and the cut of K into parts, of the fewest cycles, runs taken as equally long.  A K block costs its products (half a cycle
// for each column, 90 at least to issue one, 128 rows) or its copies (64 bytes a cycle and SM, which is where a pair of CTAs, each with half of
// the columns, gains); K is cut (the parts are added up by another launch, 6000 cycles) only where tiles are fewer than SMs.
Shape shape_of(int M, int K, int R, int runs, bool may_split) {
  const int sms = 148, each = std::max(1, (R + runs - 1) / std::max(1, runs)), nkb = (K + kBK - 1) / kBK;
  Shape best{false, 32, 1, 0};
  double least = 1e300;
  for (int pair = 0; pair <= 1; ++pair) {
    if (pair && M <= 128) break;
    for (int cap = pair ? 144 : 16; cap <= 256; cap += 16) {
      const int w = tile_width(each, cap);
      if (w != cap) continue;                          // the same tiles as a smaller cap's
      const double tiles = (double)tile_count(each, cap) * std::min(runs, R) * ((M + 127 + 128 * pair) / (128 + 128 * pair)) / (pair ? sms / 2 : sms);
      const double block = std::max(4.0 * std::max(90, w / 2) + 60, (16384 + (pair ? 64.0 : 128.0) * w) / 64);
      for (int splits = 1; splits == 1 || (may_split && !pair && splits <= 8 && tiles * splits < 1.01 && nkb / splits >= 4); ++splits) {
        const double all = tiles * splits, waves = runs == 1 ? std::ceil(all) : std::max(1.0, all + (all > 1 ? 0.5 : 0.0));
        const double cost = waves * (std::max((nkb + splits - 1) / splits * block, 3500.0 * w / 256) + 500) + (splits > 1 ? 6000 : 0);
        if (cost < least) {
          least = cost;
          best.pair = pair;
          best.cap = cap;
          best.splits = splits;
        }
      }
    }
  }
  best.cap = std::max(best.cap, 32);
  best.most = (long long)R / best.cap + std::min(R, runs) + 1;
  return best;
}

template <bool BF16>
cudaError_t fwd(const Shape& s, const Maps& m, const FwdArgs& g, cudaStream_t st) {
  if (s.pair) return launch_fwd<BF16, 256, true>(m, g, s.most, st);
  if (s.nt() == 256) return launch_fwd<BF16, 256, false>(m, g, s.most, st);
  if (s.nt() == 128) return launch_fwd<BF16, 128, false>(m, g, s.most, st);
  if (s.nt() == 64) return launch_fwd<BF16, 64, false>(m, g, s.most, st);
  return launch_fwd<BF16, 32, false>(m, g, s.most, st);
}
int box_of(const Shape& s) { return s.nt() >= 128 ? 64 : 16; }

Operand matrices(const void* p, bool trans, int M, int K, long long ld, long long stride, int count) {
  return trans ? Operand{p, K, M, ld, stride, count, nullptr, 0} : Operand{p, M, K, ld, stride, count, nullptr, 0};
}
// the columns of a product's result, gathered where they are not its own
Operand columns_of(const void* X, int K, int N, long long ld, const int* columns, int R) {
  return columns ? Operand{X, K, R, ld, 0, 1, columns, N} : Operand{X, K, N, ld, 0, 1, nullptr, 0};
}
// Whether the copy engine gathers: it takes some 65 cycles for every four columns and 64 features, for each tile of rows anew, so
// only while all columns are few; a copy of them, gathered once, costs a launch (8192 tokens twice, 14336 x 4096: 4.5 ms, 1.5 with the copy).
bool gathers_in_place(const Operand& x, const Shape& s) {
  return s.nt() <= 32 && Operand{x.p, x.wide, x.deep, x.ld, x.stride, x.count, nullptr, 0}.fits();
}

}  // namespace

static int low_step(int r) { return r <= 32 ? 32 : 64 * ((r + 63) / 64); }
int low_width(int r, int dtype) { return (dtype == NNLIB_B200_F16 ? 3 : 2) * low_step(r); }

bool grouped_umma_supports(const GroupedArgs& g, int dtype) {
  return (dtype == NNLIB_B200_F16 || dtype == NNLIB_B200_BF16) && g.M > 0 && g.K > 0 && g.N > 0 && g.R > 0 && g.G > 0 && (g.G <= kMaxRuns || !g.offsets) &&
         g.mats > 0 && encode_tiled_fn() != nullptr;
}
namespace {

size_t copies_bytes(const GroupedArgs& g, const Shape& s) {
  const Operand a = matrices(g.A, g.transA != 0, g.M, g.K, g.lda, g.strideA, g.mats), x = columns_of(g.X, g.K, g.N, g.ldx, g.columns, g.R);
  size_t n = padded(a.copy_bytes()) + (g.columns && gathers_in_place(x, s) ? 0 : padded(x.copy_bytes()));
  if (g.low.r > 0) n += padded(matrices(g.low.B, g.low.transB != 0, g.M, g.low.r, g.low.ldb, g.low.strideB, g.low.n).copy_bytes());
  return n;
}
size_t parts_bytes(const GroupedArgs& g, const Shape& s) { return padded((size_t)s.splits * g.R * g.M * sizeof(float)); }

// One product; `to` and `out`: what it writes and where.  ws: copies_bytes().  before: what of this call was launched before it (kWaitData:
// it reads that; kWaitEnd: it does not).
// odd: bytes of the pairs' matrices, read with g.low; look: the product whose pairs they are, whose matrices are looked through.
cudaError_t product(const GroupedArgs& g, int dtype, const Shape& s, int to, void* out, char* ws, int before, cudaStream_t st, unsigned char* odd = nullptr,
                    const GroupedArgs* look = nullptr) {
  bool behind = before != kWaitNone, copied = false;
  Operand a = matrices(g.A, g.transA != 0, g.M, g.K, g.lda, g.strideA, g.mats), x = columns_of(g.X, g.K, g.N, g.ldx, g.columns, g.R);
  const Runs runs{g.offsets, g.run_len, g.G, g.R};
  const bool in_place = g.columns && gathers_in_place(x, s);
  if (in_place) x = columns_of(g.X, g.K, g.N, g.ldx, nullptr, 0);
  const size_t copies = a.copy_bytes() + x.copy_bytes();
  cudaError_t e = align_operand(a, ws, g.ids || !g.offsets ? nullptr : &runs, behind, st);
  if (e == cudaSuccess) e = align_operand(x, ws, nullptr, behind, st);
  if (e != cudaSuccess) return e;
  copied = copies > 0;
  FwdArgs f;
  std::memset(&f, 0, sizeof(f));
  f.runs = runs;
  f.ids = g.ids;
  f.columns = g.columns;
  f.gather = in_place;
  f.cap = s.cap;
  f.C = out;
  f.ldc = g.ldc;
  f.scale = g.scale;
  f.scale0 = g.scale0;
  f.M = g.M; f.K = g.K; f.G = g.G; f.N = g.N; f.mats = g.mats;
  f.a_kmaj = g.transA;
  f.a_same = g.mats > 1 && g.strideA == 0;
  f.zero_rest = g.zero_rest && to == kToC;
  f.splits = s.splits;
  f.to = to;
  f.low_width = low_width(to == kToLow ? g.M : g.low.r, dtype);
  f.low_step = low_step(to == kToLow ? g.M : g.low.r);
  f.status = g.status;
  Maps m;
  if (!encode_matrix(&m.a, dtype, a, g.transA != 0) || !encode_columns(&m.x, dtype, x, in_place ? 1 : box_of(s))) return cudaErrorInvalidValue;
  m.b = m.t = m.a;
  f.vec = aligned16(out) && g.ldc % 8 == 0;
  if (g.low.r > 0 && to == kToC) {
    Operand b = matrices(g.low.B, g.low.transB != 0, g.M, g.low.r, g.low.ldb, g.low.strideB, g.low.n);
    copied = copied || b.copy_bytes() > 0;
    if ((e = align_operand(b, ws, nullptr, behind, st)) != cudaSuccess) return e;
    const Operand t{g.low.T, f.low_width, g.R, f.low_width, 0, 1, nullptr, 0};
    if (!encode_matrix(&m.b, dtype, b, g.low.transB != 0) || !encode_columns(&m.t, dtype, t, box_of(s))) return cudaErrorInvalidValue;
    f.r = g.low.r;
    f.low_same = g.low.n > 1 && g.low.strideB == 0;
  }
  const GroupedArgs* of = look ? look : f.r > 0 ? &g : nullptr;
  if (of) {
    const LowRank& l = of->low;
    f.low_runs = Runs{l.offsets, l.run_len, l.runs, of->R};
    f.low_ids = l.ids;
    f.n = l.n;
    f.low_B = l.B;
    f.low_ldb = l.ldb; f.low_strideB = l.strideB;
    f.low_kmaj = l.transB;
    f.low_T = l.T;
    f.odd = odd;
  }
  if (look) {
    f.look_r = look->low.r;
    f.look_m = look->M;
  }
  f.wait = copied ? kWaitData : before;
  return dtype == NNLIB_B200_BF16 ? fwd<true>(s, m, f, st) : fwd<false>(s, m, f, st);
}

// K is cut for few columns only: parts of many cost more than the SMs that it fills
bool few(int R, int M) { return R <= 512 && M <= 65535 * 256; }

}  // namespace

// parts: Float32 (M, R, splits); t: A X of g.low's pairs, Float32 (r, R, t_splits), or NULL
cudaError_t join_parts(const GroupedArgs& g, int dtype, int splits, const float* parts, const float* t, int t_splits, cudaStream_t st) {
  JoinArgs j;
  std::memset(&j, 0, sizeof(j));
  j.parts = parts;
  j.C = g.C;
  j.ldc = g.ldc;
  j.splits = splits; j.M = g.M; j.R = g.R; j.N = g.N; j.zero_rest = g.zero_rest;
  j.runs = Runs{g.offsets, g.run_len, g.G, g.R};
  j.columns = g.columns;
  if (t) {
    j.t = t;
    j.t_splits = t_splits; j.r = g.low.r; j.n = g.low.n; j.transB = g.low.transB;
    j.low_runs = Runs{g.low.offsets, g.low.run_len, g.low.runs, g.R};
    j.low_ids = g.low.ids;
    j.B = g.low.B;
    j.ldb = g.low.ldb; j.strideB = g.low.strideB;
    const int packet = dtype == NNLIB_B200_F32 ? 4 : 8;
    j.b_packets = aligned16(g.low.B) && g.low.ldb % packet == 0 && g.low.strideB % packet == 0 && g.low.r % packet == 0;
    j.b_pairs = reinterpret_cast<uintptr_t>(g.low.B) % (dtype == NNLIB_B200_F32 ? 8 : 4) == 0 && g.low.ldb % 2 == 0 && g.low.strideB % 2 == 0;
  }
  const dim3 grid((unsigned)g.R, (unsigned)((g.M + 255) / 256));
  count_launch();
  switch (dtype) {
    case NNLIB_B200_F16:  return launch_early(join_kernel<__half>, grid, dim3(128), 0, st, j);
    case NNLIB_B200_BF16: return launch_early(join_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, j);
    default:              return launch_early(join_kernel<float>, grid, dim3(128), 0, st, j);
  }
}
size_t grouped_umma_workspace_bytes(const GroupedArgs& g) {
  const Shape s = shape_of(g.M, g.K, g.R, g.G, few(g.R, g.M));
  return copies_bytes(g, s) + (s.splits > 1 ? parts_bytes(g, s) : 0);
}
cudaError_t grouped_umma(const GroupedArgs& g, int dtype, void* workspace, cudaStream_t st) {
  char* ws = static_cast<char*>(workspace);
  const Shape s = shape_of(g.M, g.K, g.R, g.G, few(g.R, g.M));
  if (s.splits == 1) return product(g, dtype, s, kToC, g.C, ws, kWaitNone, st);
  char* parts = ws + copies_bytes(g, s);
  const cudaError_t e = product(g, dtype, s, kToParts, parts, ws, kWaitNone, st);
  return e == cudaSuccess ? join_parts(g, dtype, s.splits, reinterpret_cast<const float*>(parts), nullptr, 0, st) : e;
}

// A X of low-rank pairs, as T or, `parts`, in Float32 parts
static Shape first_shape(const GroupedArgs& f) { return shape_of(f.M, f.K, f.R, f.G, true); }
size_t low_umma_workspace_bytes(const GroupedArgs& f) {
  const Shape s = first_shape(f);
  return copies_bytes(f, s) + (s.splits > 1 ? parts_bytes(f, s) : 0);
}
size_t low_umma_bytes(const GroupedArgs& f, int dtype) { return padded((size_t)f.R * 2 * low_width(f.M, dtype)); }
// behind: a kernel of this call is before it in the stream, whose results it does not read but whose workspace it may write
cudaError_t low_umma(const GroupedArgs& f, int dtype, void* T, void* workspace, bool behind, cudaStream_t st, unsigned char* odd, const GroupedArgs* look) {
  const int before = behind ? kWaitData : kWaitNone;
  const Shape s = first_shape(f);
  char* ws = static_cast<char*>(workspace);
  if (s.splits == 1) return product(f, dtype, s, kToLow, T, ws, before, st, odd, look);
  char* parts = ws + copies_bytes(f, s);
  const cudaError_t e = product(f, dtype, s, kToParts, parts, ws, before, st, odd, look);
  if (e != cudaSuccess) return e;
  const int width = low_width(f.M, dtype), step = low_step(f.M);
  const long long blocks = ((long long)f.R * step + 255) / 256;
  const float* p = reinterpret_cast<const float*>(parts);
  count_launch();
  const dim3 grid((unsigned)blocks);
  if (dtype == NNLIB_B200_BF16) return launch_early(join_low_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p, s.splits, f.M, f.R, static_cast<__nv_bfloat16*>(T), width, step);
  return launch_early(join_low_kernel<__half>, grid, dim3(256), 0, st, p, s.splits, f.M, f.R, static_cast<__half*>(T), width, step);
}

// W X with the pairs' term; first.R columns.  keep: T of the columns is wanted behind it (the gradients read it), at `low`.
static Shape main_shape(const GroupedArgs& m, bool keep) { return shape_of(m.M, m.K, m.R, 1, !keep && few(m.R, m.M)); }
// (a pair is read anew for each of its columns)
static bool first_by_column(const GroupedArgs& f) { return f.R <= 4 * f.G && f.K <= 64 * kLowK; }
static size_t odd_bytes(const GroupedArgs& m) { return m.low.r > 0 ? padded((size_t)m.low.n * ((m.M + 127) / 128)) : 0; }
size_t adapter_umma_workspace_bytes(const GroupedArgs& first, const GroupedArgs& m, bool keep) {
  const Shape s = main_shape(m, keep);
  if (s.splits == 1) return odd_bytes(m) + std::max(m.low.r > 0 ? low_umma_workspace_bytes(first) : 0, copies_bytes(m, s));
  Shape f = first_shape(first);
  const size_t own = copies_bytes(m, s) + parts_bytes(m, s);
  if (m.low.r == 0) return own;
  if (!first_by_column(first)) return own + copies_bytes(first, f) + parts_bytes(first, f);
  f.splits = (first.K + kLowK - 1) / kLowK;
  return own + parts_bytes(first, f);
}
cudaError_t adapter_umma(const GroupedArgs& first, GroupedArgs m, int dtype, bool keep, void* low, void* workspace, cudaStream_t st) {
  const Shape s = main_shape(m, keep);
  char* ws = static_cast<char*>(workspace);
  cudaError_t e = cudaSuccess;
  if (s.splits == 1) {
    unsigned char* odd = static_cast<unsigned char*>(workspace);
    ws += odd_bytes(m);
    if (m.low.r > 0) e = low_umma(first, dtype, low, ws, false, st, odd, &m);
    m.low.T = low;
    return e == cudaSuccess ? product(m, dtype, s, kToC, m.C, ws, m.low.r > 0 ? kWaitData : kWaitNone, st, odd) : e;
  }
  // few columns: both products in parts, joined by one launch that multiplies by B.  W X does not wait for A X, its end does.
  Shape f = first_shape(first);
  char* parts = ws + copies_bytes(m, s);
  char* rest = parts + parts_bytes(m, s);
  if (m.low.r == 0) {
    e = product(m, dtype, s, kToParts, parts, ws, kWaitNone, st);
    return e == cudaSuccess ? join_parts(m, dtype, s.splits, reinterpret_cast<const float*>(parts), nullptr, 0, st) : e;
  }
  char* of_first = rest;
  if (first_by_column(first)) {
    LowFewArgs l;
    l.A = first.A; l.X = first.X;
    l.parts = reinterpret_cast<float*>(of_first);
    l.lda = first.lda; l.strideA = first.strideA; l.ldx = first.ldx;
    l.scale = first.scale; l.scale0 = first.scale0;
    l.runs = Runs{first.offsets, first.run_len, first.G, first.R};
    l.ids = first.ids;
    l.transA = first.transA; l.r = first.M; l.K = first.K; l.R = first.R; l.mats = first.mats;
    l.vec = aligned16(first.A) && first.lda % 8 == 0 && first.strideA % 8 == 0 && (first.transA ? first.K : first.M) % 8 == 0;
    f.splits = (first.K + kLowK - 1) / kLowK;
    const dim3 grid((unsigned)first.R, (unsigned)f.splits);
    if (dtype == NNLIB_B200_BF16) low_few_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(l);
    else low_few_kernel<__half><<<grid, 256, 0, st>>>(l);
    count_launch();
    e = cudaGetLastError();
  } else {
    of_first = rest + copies_bytes(first, f);
    e = product(first, dtype, f, kToParts, of_first, rest, kWaitNone, st);
  }
  if (e == cudaSuccess) e = product(m, dtype, s, kToParts, parts, ws, kWaitEnd, st);
  return e == cudaSuccess ? join_parts(m, dtype, s.splits, reinterpret_cast<const float*>(parts), reinterpret_cast<const float*>(of_first), f.splits, st) : e;
}

// Parts of the columns that a pair's gradient is cut into: as many as there are SMs for, where that takes away 48 of a tile's blocks or more: the launch that
// adds them is some 5 us (one pair, 4096 x 16, 32768 columns: 50 us in four parts, 112 in one; 2048 columns in two parts: 4 us more than in one).
static int grad_splits(const GroupedGradArgs& g, int fold) {
  if (!fold) return 1;
  const long long tiles = (long long)(((fold == 1 ? g.K : g.M) + 127) / 128) * g.mats, blocks = g.R / 64 / g.mats;
  const long long splits = std::max<long long>(1, std::min({148 / tiles, blocks / 8, 16ll}));
  return blocks - blocks / splits < 48 ? 1 : (int)splits;
}
size_t grouped_umma_grad_workspace_bytes(const GroupedGradArgs& g, int fold) {
  const Operand c = columns_of(g.C, g.M, g.R, g.ldc, nullptr, 0), x = columns_of(g.X, g.K, g.N, g.ldx, g.columns, g.R);
  const int splits = grad_splits(g, fold);
  return (fold == 1 ? 0 : padded(c.copy_bytes())) + (fold == 2 ? 0 : padded(x.copy_bytes())) +
         (splits > 1 ? padded(sizeof(float) * splits * (size_t)g.mats * g.M * g.K) : 0);
}
bool grouped_umma_grad_supports(const GroupedGradArgs& g, int dtype) {
  return (dtype == NNLIB_B200_F16 || dtype == NNLIB_B200_BF16) && g.M > 0 && g.K > 0 && g.N > 0 && g.R > 0 && g.mats > 0 && encode_tiled_fn() != nullptr;
}
// fold: 0: none; 1: C is T, M its rank; 2: X is T, K its rank.  (The first term and what it leaves, Float16: that 2^11 times as large)
cudaError_t grouped_umma_grad(const GroupedGradArgs& g, int dtype, int fold, void* workspace, bool behind, cudaStream_t st) {
  char* ws = static_cast<char*>(workspace);
  Operand c = columns_of(g.C, fold == 1 ? low_width(g.M, dtype) : g.M, g.R, g.ldc, nullptr, 0),
          x = columns_of(g.X, fold == 2 ? low_width(g.K, dtype) : g.K, g.N, g.ldx, g.columns, g.R);
  cudaError_t e = align_operand(c, ws, nullptr, behind, st);
  if (e == cudaSuccess) e = align_operand(x, ws, nullptr, behind, st);
  if (e != cudaSuccess) return e;
  GradArgs a;
  std::memset(&a, 0, sizeof(a));
  a.runs = Runs{g.offsets, g.run_len, g.G, g.R};
  a.ids = g.ids;
  a.A = g.A;
  a.ld = g.lda; a.stride = g.strideA;
  a.G = g.G; a.mats = g.mats;
  a.status = g.status;
  a.wait = behind;
  // the folded side's terms are neighbours in a row of tensor memory; otherwise the side that is contiguous in the result is in its lanes
  const bool x_rows = fold ? fold == 1 : g.transA != 0;
  a.rows = x_rows ? g.K : g.M;
  a.cols = x_rows ? g.M : g.K;
  a.fold = fold != 0;
  a.fold_step = fold ? low_step(a.cols) : 0;
  a.fold_at = dtype == NNLIB_B200_F16 ? a.fold_step : 0;
  a.fold_scale = dtype == NNLIB_B200_F16 ? 1.f / kScaled : 1.f;
  a.along = fold && (fold == 1) == (g.transA == 0);
  const int nt = fold ? 2 * a.fold_step : 256;
  const bool pair = !fold && a.rows > 128 && a.cols > 128;
  CUtensorMap mc, mx;
  if (!encode_columns(&mc, dtype, c, 64) || !encode_columns(&mx, dtype, x, 64)) return cudaErrorInvalidValue;
  a.vec = aligned16(g.A) && g.lda % 8 == 0 && g.strideA % 8 == 0;
  const CUtensorMap& r = x_rows ? mx : mc;
  const CUtensorMap& q = x_rows ? mc : mx;
  const bool bf16 = dtype == NNLIB_B200_BF16;
  a.splits = grad_splits(g, fold);
  if (a.splits > 1) a.parts = reinterpret_cast<float*>(ws);       // (behind the copies)
  auto run = [&] {
    if (pair) return bf16 ? launch_bwd<true, 256, true>(r, q, a, st) : launch_bwd<false, 256, true>(r, q, a, st);
    if (nt == 256) return bf16 ? launch_bwd<true, 256, false>(r, q, a, st) : launch_bwd<false, 256, false>(r, q, a, st);
    if (nt == 128) return bf16 ? launch_bwd<true, 128, false>(r, q, a, st) : launch_bwd<false, 128, false>(r, q, a, st);
    return bf16 ? launch_bwd<true, 64, false>(r, q, a, st) : launch_bwd<false, 64, false>(r, q, a, st);
  };
  if ((e = run()) != cudaSuccess || !a.parts) return e;
  JoinGradArgs j;
  std::memset(&j, 0, sizeof(j));
  j.parts = a.parts;
  j.A = a.A;
  j.ld = a.ld; j.stride = a.stride;
  j.rows = a.rows; j.cols = a.cols; j.mats = a.mats; j.splits = a.splits; j.along = a.along;
  count_launch();
  const dim3 grid((unsigned)((a.rows + 31) / 32), (unsigned)a.mats);
  return bf16 ? launch_early(join_grad_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, j) : launch_early(join_grad_kernel<__half>, grid, dim3(256), 0, st, j);
}

// Reads and clears the sticky "a bounded wait ran out" flag of these kernels on the current device.
cudaError_t grouped_take_abort(int* out, cudaStream_t st) {
  int v = 0;
  cudaError_t e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return e;
  e = cudaMemcpyFromSymbol(&v, g_grouped_abort, sizeof(int));
  if (e != cudaSuccess) return e;
  if (v) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_grouped_abort, &zero, sizeof(int));
  }
  *out = v;
  return e;
}

}  // namespace nb200
