// Products of ragged groups of columns on the CUDA cores, products and sums in fp32, any element type, size and stride: Float32 arrays, and
// what of the 16-bit ones grouped_umma.cu does not take.
//
//   grouped_fma_kernel     C[:, i] = A_g X[:, columns[i]] for the columns i of run g, and, for low-rank pairs, + B_a T[:, i]
//   grouped_narrow_kernel  the same for runs of up to four columns
//   grouped_grad_kernel    A_a = sum over the columns i of the runs of matrix a of C[:, i] X[:, columns[i]]^T
//
// 256 threads compute 128 rows x BN columns, k in steps of 16 or 32 through two shared-memory stages [k][row]: while one is multiplied the next
// one's elements are on their way into registers, four neighbours at a time.  A thread multiplies 8 rows and 8 columns as packed pairs of
// rows, in narrow tiles of every 128 / BN-th k.  A block's slot number is turned into (run, first column) by counting the tiles of all runs, since their sizes
// are on the device only; slots that no run needs end at once.  Few tiles: K is cut and the parts are added by another launch (join_parts).
// What bounds it: the FMA pipe and the shared memory that feeds it where columns are many (2048 x 2048, 4096 columns in 8 runs: 822 us,
// 42 TFLOP/s, with two blocks to an SM and 128 registers; 883 with one; the gradient of the matrices 802 and 1086), reading A where they are few (6248 x 6680, 64 columns in 3 runs: 288 us, 1.7 TB/s).
// (Of these, 15 and 10 us are what the compiler makes of 128 registers since a block also sees to columns in no run where offsets fall.)
#include <algorithm>

#include "common.cuh"
#include "grouped_runs.cuh"
#include "launchers.h"
#include "umma.cuh"

namespace nb200 {
namespace {

using ptx::pair_add;
using ptx::pair_fma;
using ptx::pair_of;
using ptx::pair_unpack;

constexpr int kRows = 128;                   // rows to a tile

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
    return make_float4(Elem<T>::to_f(e[0]), Elem<T>::to_f(e[1]), Elem<T>::to_f(e[2]), Elem<T>::to_f(e[3]));
  }
}

// One side of a contraction: elements (k, r) of W rows r, as they lie in memory.
//   along:  k contiguous; row r begins at base + row(r) * ld, or is none (row(r) < 0: zeros)
//   else    r contiguous; step k begins at base + step(k) * ld, or is none (zeros); `rows` of them are there
template <typename T>
struct Side {
  const T* base;
  long long ld;
  bool along, vec;                           // vec: four neighbours at an address of their size's multiple
  int rows;
  const int* table;                          // along: row(r), in shared memory, or NULL: r < rows; else step(k) of the whole contraction, or NULL: k
  int limit;                                 // else, with a table: its entries below this are there
};

// k to a stage: the narrowest tiles are there to read A, 16 KB of it at a time (of 32 columns: 309 us instead of 295, spilled)
__host__ __device__ constexpr int step_of(int bn) { return bn <= 16 ? 32 : 16; }

template <typename T, int W, int KS>
struct Loader {
  static constexpr int NV = W * KS >= 1024 ? W * KS / 1024 : 1, kThreads = W * KS / 4 / NV;   // of 256 threads, these load
  const Side<T>& s;
  float4 v[NV];
  __device__ __forceinline__ Loader(const Side<T>& side) : s(side) {}
  __device__ __forceinline__ void fetch(int k0, int K) {
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int q = threadIdx.x + 256 * e;
      v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (kThreads < 256 && threadIdx.x >= kThreads) continue;
      float* f = reinterpret_cast<float*>(&v[e]);
      if (s.along) {
        const int k = k0 + (q % (KS / 4)) * 4, r = q / (KS / 4), row = s.table ? s.table[r] : (r < s.rows ? r : -1);
        if (row < 0) continue;
        const T* p = s.base + row * s.ld + k;
        if (s.vec && k + 4 <= K) {
          v[e] = load4(p);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k + i < K) f[i] = Elem<T>::to_f(p[i]);
        }
      } else {
        const int r = (q % (W / 4)) * 4, k = k0 + q / (W / 4);
        if (k >= K || r >= s.rows) continue;
        const int step = s.table ? s.table[k] : k;
        if (s.table && (unsigned)step >= (unsigned)s.limit) continue;
        const T* p = s.base + step * s.ld + r;
        if (s.vec && r + 4 <= s.rows) {
          v[e] = load4(p);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + i < s.rows) f[i] = Elem<T>::to_f(p[i]);
        }
      }
    }
  }
  __device__ __forceinline__ void stage(float (*t)[W + 4]) {
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int q = threadIdx.x + 256 * e;
      if (kThreads < 256 && threadIdx.x >= kThreads) continue;
      if (s.along) {
        const int k = (q % (KS / 4)) * 4, r = q / (KS / 4);
        t[k][r] = v[e].x;
        t[k + 1][r] = v[e].y;
        t[k + 2][r] = v[e].z;
        t[k + 3][r] = v[e].w;
      } else {
        *reinterpret_cast<float4*>(&t[q / (W / 4)][(q % (W / 4)) * 4]) = v[e];
      }
    }
  }
};

// A thread's part of a 128 x BN tile: 8 rows row(j) and 8 columns, of every kParts-th k, so that a step's four 16-byte reads of shared memory feed 64
// products whatever the tile is (with 8 x 2 of every k tiles of 32 columns took 378 us where these take 277: 6248 x 6680,
// 64 columns in 3 runs).  join()
// adds the parts, in their order; then the thread has all of k for kOwn columns, column(i).
template <int BN>
struct Tile {
  static constexpr int kParts = 128 / BN, kOwn = 8 / kParts, kLanes = 256 / kParts;
  static constexpr int kJoin = kParts > 1 ? 4 * kOwn * (kParts - 1) * kLanes : 1;      // pairs of rows that join() has in shared memory
  unsigned long long acc[8][4], own[kParts > 1 ? kOwn : 1][4];              // pairs of rows
  static __device__ __forceinline__ int part() { return threadIdx.x / kLanes; }
  static __device__ __forceinline__ int lane() { return threadIdx.x % kLanes; }
  // a warp's lanes: 8 fours of rows by 4 fours of columns
  static __device__ __forceinline__ int tx() { return BN > 16 ? (lane() & 7) + ((lane() >> 5) & 1) * 8 : lane() & 15; }
  static __device__ __forceinline__ int ty() { return BN > 16 ? ((lane() >> 3) & 3) + (lane() >> 6) * 4 : lane() >> 4; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0ull;
  }
  __device__ __forceinline__ void step(const float* p, const float* q) {
    unsigned long long a[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p + tx() * 4 + h * 64);
      a[2 * h] = v.x;
      a[2 * h + 1] = v.y;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 v = *reinterpret_cast<const float4*>(q + ty() * 4 + h * (BN / 2));
      const float b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned long long bb = pair_of(b[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[h * 4 + i][j] = pair_fma(a[j], bb, acc[h * 4 + i][j]);
      }
    }
  }
  // by the whole block, behind a barrier; leaves one behind itself
  __device__ __forceinline__ void join(unsigned long long* room) {
    if constexpr (kParts > 1) {
      const int me = part(), t = lane();
#pragma unroll
      for (int d = 0; d < kParts; ++d) {
        if (me != d) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) room[((i * 4 + j) * (kParts - 1) + me - (me > d ? 1 : 0)) * kLanes + t] = acc[d * kOwn + i][j];
        }
        __syncthreads();
        if (me == d) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              // (part 0 first, whoever adds: a column's sum is the same in every place)
              auto part_of = [&](int q) { return q == d ? acc[d * kOwn + i][j] : room[((i * 4 + j) * (kParts - 1) + q - (q > d ? 1 : 0)) * kLanes + t]; };
              unsigned long long v = part_of(0);
#pragma unroll
              for (int q = 1; q < kParts; ++q) v = pair_add(v, part_of(q));
              own[i][j] = v;
            }
        }
        __syncthreads();
      }
    }
  }
  __device__ __forceinline__ void values(int i, float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) pair_unpack(kParts > 1 ? own[kParts > 1 ? i : 0][j] : acc[i][j], v[2 * j], v[2 * j + 1]);
  }
  static __device__ __forceinline__ int row(int j) { return tx() * 4 + (j >> 2) * 64 + (j & 3); }
  static __device__ __forceinline__ int column(int i) {
    const int c = part() * kOwn + i;
    return ty() * 4 + (c >> 2) * (BN / 2) + (c & 3);
  }
};

template <int BN>
struct Stages {
  static constexpr int kStep = step_of(BN);
  float p[2][kStep][kRows + 4], q[2][kStep][BN + 4];
};
template <int BN>
union alignas(16) Shared {
  Stages<BN> stages;
  unsigned long long joined[Tile<BN>::kJoin];
};

// One contraction over k0 .. K - 1 (k0 a multiple of 4)
template <int BN, typename TP, typename TQ>
__device__ __forceinline__ void contract(Tile<BN>& t, Stages<BN>& s, int k0, int K, const Side<TP>& P, const Side<TQ>& Q) {
  constexpr int kStep = step_of(BN);
  if (K <= k0) return;
  Loader<TP, kRows, kStep> p(P);
  Loader<TQ, BN, kStep> q(Q);
  p.fetch(k0, K);
  q.fetch(k0, K);
  __syncthreads();                           // (an earlier contraction's last stage has been read)
  p.stage(s.p[0]);
  q.stage(s.q[0]);
  __syncthreads();
  for (int b = 0; k0 < K; k0 += kStep, b ^= 1) {
    const bool more = k0 + kStep < K;
    if (more) {
      p.fetch(k0 + kStep, K);
      q.fetch(k0 + kStep, K);
    }
    const int kn = min(kStep, K - k0);       // the padding is not multiplied: 0 * Inf would be a NaN
    if (kn == kStep) {
#pragma unroll
      for (int k = 0; k < kStep; k += Tile<BN>::kParts) t.step(s.p[b][k + Tile<BN>::part()], s.q[b][k + Tile<BN>::part()]);
    } else {
      for (int k = Tile<BN>::part(); k < kn; k += Tile<BN>::kParts) t.step(s.p[b][k], s.q[b][k]);
    }
    if (more) {
      p.stage(s.p[b ^ 1]);
      q.stage(s.q[b ^ 1]);
    }
    __syncthreads();
  }
}

template <typename T>
__host__ __device__ __forceinline__ bool fours(const T* p, long long a, long long b) {
  return (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0 && a % 4 == 0 && b % 4 == 0;
}

// blockIdx: (slot of columns, tile of rows, part of K).  parts: Float32 (M, R, parts) instead of C
template <typename T, typename TC, int BN>
__global__ void __launch_bounds__(256, 2) grouped_fma_kernel(const __grid_constant__ GroupedArgs g, float* parts) {
  __shared__ Shared<BN> shared;
  Stages<BN>& st = shared.stages;
  __shared__ RunSearch search;
  __shared__ int cols[BN];
  const Runs runs{g.offsets, g.run_len, g.G, g.R};
  const RunTile run = find_run(runs, g.zero_rest && !parts, BN, blockIdx.x, gridDim.x, search);
  if (run.run == kNoRun) return;
  const int m0 = blockIdx.y * kRows, n0 = run.first, nn = min(BN, run.end - n0);
  if (run.run == kScattered) {
    clear_scattered(runs, run, reinterpret_cast<TC*>(g.C), g.ldc, m0, min(kRows, g.M - m0), search);
    return;
  }
  const int mat = run.run < 0 ? -1 : (g.ids ? g.ids[run.run] : run.run);
  const bool have = mat >= 0 && mat < g.mats;
  for (int i = threadIdx.x; i < BN; i += 256) {
    int c = -1;
    if (have && i < nn) {
      c = g.columns ? g.columns[n0 + i] : n0 + i;
      if (c < 0 || c >= g.N) c = -1;
    }
    cols[i] = c;
  }
  __syncthreads();
  Tile<BN> t;
  t.clear();
  const int rows = min(kRows, g.M - m0);
  if (have) {
    const T* A = reinterpret_cast<const T*>(g.A) + (long long)mat * g.strideA + (g.transA ? (long long)m0 * g.lda : m0);
    const T* X = reinterpret_cast<const T*>(g.X);
    const int each = ((g.K + gridDim.z - 1) / gridDim.z + 31) / 32 * 32, k0 = blockIdx.z * each;
    contract<BN>(t, st, k0, min(g.K, k0 + each), Side<T>{A, g.lda, g.transA != 0, fours(A, g.lda, 0), rows, nullptr, 0},
                 Side<T>{X, g.ldx, true, fours(X, g.ldx, 0), BN, cols, 0});
  }
  t.join(shared.joined);
  const float scale = !have ? 0.f : (g.scale ? g.scale[mat] : g.scale0);
  float c[Tile<BN>::kOwn][8];
#pragma unroll
  for (int i = 0; i < Tile<BN>::kOwn; ++i) {
    t.values(i, c[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) c[i][j] *= scale;
  }
  if (g.low.r > 0) {
    // The runs of pairs that have columns here, one after the other; columns of other runs take no part.  Of 256 runs the block sees in one go whether
    // any has, of equal ones it begins with the first that has (20000 single columns, 256 x 256: 3020 us; 9940 where each block goes through all).
    const Runs of{g.low.offsets, g.low.run_len, g.low.runs, g.R};
    const float* low = reinterpret_cast<const float*>(g.low.T);
    __shared__ int mine[BN];
    const int b0 = of.offsets ? 0 : of.len > 0 ? (int)min((long long)of.runs, n0 / of.len) : of.runs;
    for (int b = b0; b < of.runs; ++b) {
      if (((b - b0) & 255) == 0) {
        const auto meets = [&](int i) { return i < of.runs && max(of.begin(i), n0) < min(of.end(i), n0 + nn); };
        while (b < of.runs && !__syncthreads_or(meets(b + (int)threadIdx.x))) b = of.offsets ? b + 256 : of.runs;
        if (b >= of.runs) break;
      }
      const int lo = max(of.begin(b), n0), hi = min(of.end(b), n0 + nn), id = g.low.ids[b];
      if (lo >= hi || id < 0 || id >= g.low.n) continue;
      const T* B = reinterpret_cast<const T*>(g.low.B) + (long long)id * g.low.strideB + (g.low.transB ? (long long)m0 * g.low.ldb : m0);
      __syncthreads();
      for (int i = threadIdx.x; i < BN; i += 256) mine[i] = n0 + i >= lo && n0 + i < hi ? n0 + i : -1;
      __syncthreads();
      t.clear();
      contract<BN>(t, st, 0, g.low.r, Side<T>{B, g.low.ldb, g.low.transB != 0, fours(B, g.low.ldb, 0), rows, nullptr, 0},
                   Side<float>{low, g.low.ldt, true, fours(low, g.low.ldt, 0), BN, mine, 0});
      t.join(shared.joined);
#pragma unroll
      for (int i = 0; i < Tile<BN>::kOwn; ++i) {
        const int n = n0 + Tile<BN>::column(i);
        if (n < lo || n >= hi) continue;     // (0 * Inf of another pair's matrix)
        float v[8];
        t.values(i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) c[i][j] += v[j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < Tile<BN>::kOwn; ++i) {
    const int n = Tile<BN>::column(i);
    if (n >= nn) continue;
    const bool zero = cols[n] < 0;           // (a padding column's 0 times an infinity of A)
    if (parts) {
      float* out = parts + ((long long)blockIdx.z * g.R + n0 + n) * g.M + m0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (Tile<BN>::row(j) < rows) out[Tile<BN>::row(j)] = c[i][j];
    } else {
      TC* out = reinterpret_cast<TC*>(g.C) + (long long)(n0 + n) * g.ldc + m0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (Tile<BN>::row(j) < rows) out[Tile<BN>::row(j)] = Elem<TC>::from_f(zero ? 0.f : c[i][j]);
    }
  }
}

// Runs of a few columns: nothing of A is read twice, so none of it goes through shared memory.  128 rows and up to kNarrow columns to a block.
// Rows contiguous: a lane has four rows, every eighth k is a warp's; k contiguous: a warp has 16 rows, a lane every 32nd four of k.
// (two columns to each of 128 matrices of 1536 x 2048: 427 us, 3.8 TB/s, turned; 512 us not; in tiles of 16 columns 1148 us)
constexpr int kNarrow = 4, kChunk = 1024;
template <typename T, typename TC, bool TURNED>
__global__ void __launch_bounds__(256, TURNED ? 2 : 3) grouped_narrow_kernel(const __grid_constant__ GroupedArgs g, float* parts) {
  __shared__ __align__(16) float x[kNarrow][kChunk];
  __shared__ __align__(16) float sums[8][kNarrow][kRows];
  __shared__ RunSearch search;
  const Runs runs{g.offsets, g.run_len, g.G, g.R};
  const RunTile run = find_run(runs, g.zero_rest && !parts, kNarrow, blockIdx.x, gridDim.x, search);
  if (run.run == kNoRun) return;
  const int m0 = blockIdx.y * kRows, n0 = run.first, nn = min(kNarrow, run.end - n0), rows = min(kRows, g.M - m0);
  if (run.run == kScattered) {
    clear_scattered(runs, run, reinterpret_cast<TC*>(g.C), g.ldc, m0, rows, search);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mat = run.run < 0 ? -1 : (g.ids ? g.ids[run.run] : run.run);
  const bool have = mat >= 0 && mat < g.mats;
  int col[kNarrow];
#pragma unroll
  for (int c = 0; c < kNarrow; ++c) {
    col[c] = have && c < nn ? (g.columns ? g.columns[n0 + c] : n0 + c) : -1;
    if (col[c] >= g.N) col[c] = -1;
  }
  constexpr int kMine = TURNED ? 16 : 4;
  float acc[kMine][kNarrow];
#pragma unroll
  for (int i = 0; i < kMine; ++i)
#pragma unroll
    for (int c = 0; c < kNarrow; ++c) acc[i][c] = 0.f;
  const int each = ((g.K + gridDim.z - 1) / gridDim.z + 31) / 32 * 32, k1 = have ? min(g.K, (int)(blockIdx.z + 1) * each) : 0;
  const T* A = reinterpret_cast<const T*>(g.A) + (long long)(have ? mat : 0) * g.strideA + (TURNED ? (long long)m0 * g.lda : m0);
  const bool vec = fours(A, g.lda, 0);
  for (int k0 = blockIdx.z * each; k0 < k1; k0 += kChunk) {
    const int nk = min(kChunk, k1 - k0);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kNarrow; ++c)
      for (int k = threadIdx.x; k < nk; k += 256)
        x[c][k] = col[c] >= 0 ? Elem<T>::to_f(reinterpret_cast<const T*>(g.X)[(long long)col[c] * g.ldx + k0 + k]) : 0.f;
    __syncthreads();
    if constexpr (!TURNED) {
      const int r = lane * 4;
      const T* a = A + (long long)k0 * g.lda + r;
#pragma unroll 8
      for (int k = warp; k < nk; k += 8) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const T* p = a + (long long)k * g.lda;
        if (vec && r + 4 <= rows) {
          const float4 f = load4(p);
          v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + i < rows) v[i] = Elem<T>::to_f(p[i]);
        }
#pragma unroll
        for (int c = 0; c < kNarrow; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][c] = fmaf(v[i], x[c][k], acc[i][c]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {          // four rows at a time
#pragma unroll 2
        for (int k = lane * 4; k < nk; k += 128) {
          float4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = warp * 16 + q * 4 + i;
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r >= rows) continue;
            const T* p = A + r * g.lda + k0 + k;
            if (vec && k + 4 <= nk) {
              v[i] = load4(p);
            } else {
              float* f = reinterpret_cast<float*>(&v[i]);
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (k + u < nk) f[u] = Elem<T>::to_f(p[u]);
            }
          }
#pragma unroll
          for (int c = 0; c < kNarrow; ++c) {
            float4 b = *reinterpret_cast<const float4*>(&x[c][k]);
            if (k + 4 > nk) {                // (what is behind the end of the chunk is an older one's)
              if (k + 1 >= nk) b.y = 0.f;
              if (k + 2 >= nk) b.z = 0.f;
              b.w = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[q * 4 + i][c] = fmaf(v[i].x, b.x, fmaf(v[i].y, b.y, fmaf(v[i].z, b.z, fmaf(v[i].w, b.w, acc[q * 4 + i][c]))));
          }
        }
      }
    }
  }
  // to sums[w][c][row]: w = 8 warps of every row, or one
  if constexpr (!TURNED) {
#pragma unroll
    for (int c = 0; c < kNarrow; ++c) *reinterpret_cast<float4*>(&sums[warp][c][lane * 4]) = make_float4(acc[0][c], acc[1][c], acc[2][c], acc[3][c]);
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int c = 0; c < kNarrow; ++c) {
        float v = acc[i][c];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) sums[0][c][warp * 16 + i] = v;
      }
  }
  __syncthreads();
  const float scale = !have ? 0.f : (g.scale ? g.scale[mat] : g.scale0);
  for (int i = threadIdx.x; i < kNarrow * kRows; i += 256) {
    const int c = i / kRows, r = i % kRows;
    if (c >= nn || r >= rows) continue;
    float v = sums[0][c][r];
    if (!TURNED)
      for (int w = 1; w < 8; ++w) v += sums[w][c][r];
    v *= scale;
    if (parts) parts[((long long)blockIdx.z * g.R + n0 + c) * g.M + m0 + r] = v;
    else {
      const int from = have ? (g.columns ? g.columns[n0 + c] : n0 + c) : -1;
      reinterpret_cast<TC*>(g.C)[(long long)(n0 + c) * g.ldc + m0 + r] = Elem<TC>::from_f((unsigned)from < (unsigned)g.N ? v : 0.f);
    }
  }
}

// blockIdx: (tile of A's shorter way, tile of its contiguous one, matrix).  The tile's rows are those along which A is contiguous, so that it is
// stored in long pieces: C's rows, or, turned, X's.  (64 columns in 3 runs, 6248 x 6680, turned: 210 us; 298 with one block to an SM; 558 with that and C's rows)
template <typename TP, typename TQ, typename TA, int BN>
__global__ void __launch_bounds__(256, 2) grouped_grad_kernel(const __grid_constant__ GroupedGradArgs g) {
  __shared__ Shared<BN> shared;
  Stages<BN>& st = shared.stages;
  const bool turned = g.transA != 0;
  const int P = turned ? g.K : g.M, Q = turned ? g.M : g.K;
  const int q0 = blockIdx.x * BN, p0 = blockIdx.y * kRows, a = blockIdx.z, rows = min(kRows, P - p0), cols = min(BN, Q - q0);
  const void *p_base = turned ? g.X : g.C, *q_base = turned ? g.C : g.X;
  const long long ldp = turned ? g.ldx : g.ldc, ldq = turned ? g.ldc : g.ldx;
  const Runs of{g.offsets, g.run_len, g.G, g.R};
  Tile<BN> t;
  t.clear();
  // the runs of matrix a: a warp looks at 32 at a time, and every warp finds the same
  int b = g.ids ? -1 : a - 1, at = -32;
  unsigned found = 0u;
  while (true) {
    if (!g.ids) {
      if (++b > a || b >= g.G) break;
    } else {
      while (found == 0u && (at += 32) < g.G) {
        const int i = at + (int)(threadIdx.x & 31);
        found = __ballot_sync(0xffffffffu, i < g.G && g.ids[i] == a);
      }
      if (found == 0u) break;
      b = at + __ffs(found) - 1;
      found &= found - 1u;
    }
    const int lo = of.begin(b), n = of.end(b) - lo;
    const int* table = g.columns ? g.columns + lo : nullptr;
    const int *p_table = turned ? table : nullptr, *q_table = turned ? nullptr : table;
    const TP* p = reinterpret_cast<const TP*>(p_base) + (p_table ? 0 : (long long)lo * ldp) + p0;
    const TQ* q = reinterpret_cast<const TQ*>(q_base) + (q_table ? 0 : (long long)lo * ldq) + q0;
    contract<BN>(t, st, 0, n, Side<TP>{p, ldp, false, fours(p, ldp, 0), rows, p_table, g.N}, Side<TQ>{q, ldq, false, fours(q, ldq, 0), cols, q_table, g.N});
  }
  t.join(shared.joined);
  TA* A = reinterpret_cast<TA*>(g.A) + (long long)a * g.strideA + p0;
  const bool vec = fours(A, g.lda, 0);
#pragma unroll
  for (int i = 0; i < Tile<BN>::kOwn; ++i) {
    const int c = Tile<BN>::column(i);
    if (c >= cols) continue;
    float v[8];
    t.values(i, v);
    TA* out = A + (long long)(q0 + c) * g.lda;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      const int r = Tile<BN>::row(h);
      if (vec && sizeof(TA) == 4 && r + 4 <= rows) {
        *reinterpret_cast<float4*>(out + r) = make_float4(v[h], v[h + 1], v[h + 2], v[h + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r + j < rows) out[r + j] = Elem<TA>::from_f(v[h + j]);
      }
    }
  }
}

struct FmaShape {
  int bn, splits;
};
// As many columns to a tile as the average run has (64 instead of 128 where that pads a tenth less: 8107 x 6384 by 165 columns 561 us, 620 of 128),
// fewer where that leaves SMs without a tile (333 x 200 by 1200 columns in 5 runs: 36 us
// in tiles of 128 columns, 19 us of 32), and K cut into parts of at least 128, while these are few, where full waves of blocks gain a tenth by it: a block costs its k and
// some 96 more, the launch that adds the parts about 50 k (6680 x 6248 by 64 columns in 3 runs, 159 blocks: 432 us in 2 parts, 309 in more).
FmaShape fma_shape(const GroupedArgs& g) {
  const long long each = std::max<long long>(1, g.R / std::max(1, g.G)), rows = (g.M + kRows - 1) / kRows;
  FmaShape s;
  auto padded = [&](int bn) { return (each + bn - 1) / bn * bn; };
  s.bn = each > 64 ? (10 * padded(64) < 9 * padded(128) ? 64 : 128) : each > 32 ? 64 : each > 16 ? 32 : each > kNarrow ? 16 : kNarrow;
  auto tiles = [&] { return ((each + s.bn - 1) / s.bn) * std::min(g.G, g.R) * rows; };
  auto cut = [&] {
    const long long slots = 296;
    long long least = 0;
    int best = 1;
    for (int n = 1; n <= 32 && (n == 1 || g.K / n >= 128); n *= 2) {
      if (n > 1 && g.R > 512 && 8ll * n * g.R * g.M > (32ll << 20)) break;
      const long long cost = ((tiles() * n + slots - 1) / slots) * (g.K / n + 96) + (n > 1 ? 40 + 8 * n : 0);
      if (n == 1 || 10 * cost < 9 * least) { least = cost; best = n; }
    }
    return best;
  };
  while (s.bn > 32 && tiles() * cut() < 148) s.bn /= 2;
  s.splits = cut();
  if (s.bn == kNarrow && g.low.r > 0 && s.splits == 1) s.bn = 16;      // (low-rank pairs: in the wider tiles, or by the launch that adds the parts)
  return s;
}

template <typename T, typename TC>
cudaError_t launch_of(const GroupedArgs& g, const FmaShape& s, float* parts, cudaStream_t st) {
  const long long slots = run_slots(g.R, g.G, s.bn), rows = (g.M + kRows - 1) / kRows;
  if (slots > 0x7fffffffLL || rows > 65535) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)slots, (unsigned)rows, (unsigned)s.splits);
  switch (s.bn) {
    case 128: grouped_fma_kernel<T, TC, 128><<<grid, 256, 0, st>>>(g, parts); break;
    case 64:  grouped_fma_kernel<T, TC, 64><<<grid, 256, 0, st>>>(g, parts); break;
    case 32:  grouped_fma_kernel<T, TC, 32><<<grid, 256, 0, st>>>(g, parts); break;
    case 16:  grouped_fma_kernel<T, TC, 16><<<grid, 256, 0, st>>>(g, parts); break;
    default:
      if (g.transA) grouped_narrow_kernel<T, TC, true><<<grid, 256, 0, st>>>(g, parts);
      else grouped_narrow_kernel<T, TC, false><<<grid, 256, 0, st>>>(g, parts);
      break;
  }
  count_launch();
  return cudaGetLastError();
}

template <typename TP, typename TQ, typename TA>
cudaError_t launch_grad_tiles(const GroupedGradArgs& g, cudaStream_t st) {
  const long long P = g.transA ? g.K : g.M, Q = g.transA ? g.M : g.K, rows = (P + kRows - 1) / kRows;
  if (rows > 65535 || g.mats > 65535) return cudaErrorInvalidConfiguration;
  auto blocks = [&](long long bn) { return ((Q + bn - 1) / bn) * rows * g.mats; };
  const int bn = Q > 64 && blocks(128) >= 148 ? 128 : Q > 32 && blocks(64) >= 148 ? 64 : Q > 16 ? 32 : 16;
  const dim3 grid((unsigned)((Q + bn - 1) / bn), (unsigned)rows, (unsigned)g.mats);
  switch (bn) {
    case 128: grouped_grad_kernel<TP, TQ, TA, 128><<<grid, 256, 0, st>>>(g); break;
    case 64:  grouped_grad_kernel<TP, TQ, TA, 64><<<grid, 256, 0, st>>>(g); break;
    case 32:  grouped_grad_kernel<TP, TQ, TA, 32><<<grid, 256, 0, st>>>(g); break;
    default:  grouped_grad_kernel<TP, TQ, TA, 16><<<grid, 256, 0, st>>>(g); break;
  }
  count_launch();
  return cudaGetLastError();
}
template <typename TC, typename TX, typename TA>
cudaError_t launch_grad_of(const GroupedGradArgs& g, cudaStream_t st) {
  if (g.M < 1 || g.K < 1 || g.mats < 1) return cudaSuccess;
  return g.transA ? launch_grad_tiles<TX, TC, TA>(g, st) : launch_grad_tiles<TC, TX, TA>(g, st);
}

}  // namespace

// parts: Float32 (M, R, grouped_fma_splits(g)) instead of C
int grouped_fma_splits(const GroupedArgs& g) { return fma_shape(g).splits; }
cudaError_t grouped_fma(const GroupedArgs& g, int dtype, bool f32_out, float* parts, cudaStream_t st) {
  if (g.M < 1 || g.R < 1) return cudaSuccess;
  FmaShape s = fma_shape(g);
  if (!parts) s.splits = 1;
  switch (dtype) {
    case NNLIB_B200_F16:  return f32_out ? launch_of<__half, float>(g, s, parts, st) : launch_of<__half, __half>(g, s, parts, st);
    case NNLIB_B200_BF16: return f32_out ? launch_of<__nv_bfloat16, float>(g, s, parts, st) : launch_of<__nv_bfloat16, __nv_bfloat16>(g, s, parts, st);
    default:              return launch_of<float, float>(g, s, parts, st);
  }
}
// f32_rows / f32_cols: C / X are Float32, whatever A is
cudaError_t grouped_fma_grad(const GroupedGradArgs& g, int dtype, bool f32_rows, bool f32_cols, cudaStream_t st) {
  switch (dtype) {
    case NNLIB_B200_F16:
      return f32_rows ? launch_grad_of<float, __half, __half>(g, st) : f32_cols ? launch_grad_of<__half, float, __half>(g, st)
                                                                               : launch_grad_of<__half, __half, __half>(g, st);
    case NNLIB_B200_BF16:
      return f32_rows ? launch_grad_of<float, __nv_bfloat16, __nv_bfloat16>(g, st)
                      : f32_cols ? launch_grad_of<__nv_bfloat16, float, __nv_bfloat16>(g, st)
                                 : launch_grad_of<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(g, st);
    default: return launch_grad_of<float, float, float>(g, st);
  }
}

}  // namespace nb200
