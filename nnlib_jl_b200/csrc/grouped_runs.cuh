// Runs of columns whose ends are on the device: what a block does to find the tile that is its own.
#pragma once

#include <cuda_runtime.h>

namespace nb200 {
namespace {

constexpr int kRest = -1;                // a tile of columns in no run, before the first or behind the last
constexpr int kNoRun = -2;               // no tile at all
constexpr int kScattered = -3;           // offsets fall somewhere: what columns are in no run is seen column by column

struct Runs {
  const int* offsets;                    // (runs + 1); NULL: len columns each
  long long len;
  int runs, R;                           // R: columns there are
  __device__ __forceinline__ int at(int i) const {
    const long long o = offsets ? (long long)offsets[i] : len * i;
    return (int)(o < 0 ? 0 : (o > R ? R : o));
  }
  __device__ __forceinline__ int begin(int i) const { return at(i); }
  __device__ __forceinline__ int end(int i) const { return max(at(i), at(i + 1)); }
};

struct RunTile {
  int run, first, end;                   // the tile begins at column `first` of a run (or rest) that ends before `end`
};
struct RunSearch {
  int part[32];
  RunTile found;
};

// Tile number `slot` of `slots` when the columns of every run in turn, before the first one and behind the last one (rest) are
// cut into tiles of bt columns.  Where offsets fall, the slots behind the runs' tiles are {kScattered, number, how many}.  Called by a whole block of whole warps.
__device__ inline RunTile find_run(const Runs& of, bool rest, int bt, int slot, int slots, RunSearch& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int carry = 0;
  bool falls = false;
  for (int i0 = 0; i0 < of.runs; i0 += blockDim.x) {
    const int i = i0 + (int)threadIdx.x;
    int first = 0, end = 0;
    if (i < of.runs) {
      first = of.begin(i);
      end = of.end(i);
      falls = falls || (rest && of.at(i + 1) < first);
    }
    const int own = end > first ? (end - first + bt - 1) / bt : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (lane == 31) s.part[warp] = sum;
    __syncthreads();
    int before = carry, all = carry;
    for (int q = 0; q < warps; ++q) {
      if (q < warp) before += s.part[q];
      all += s.part[q];
    }
    const int at = slot - (before + sum - own);
    if (at >= 0 && at < own) s.found = {i, first + at * bt, end};
    carry = all;
    __syncthreads();
    if (slot < carry) return s.found;    // (the same for every thread)
  }
  if (!rest) return {kNoRun, 0, 0};
  if (__syncthreads_or(falls)) return {kScattered, slot - carry, slots - carry};
  const int first = of.runs > 0 ? of.at(0) : of.R, last = of.runs > 0 ? of.at(of.runs) : of.R, before = (first + bt - 1) / bt;
  if (slot - carry < before) return {kRest, (slot - carry) * bt, first};
  const long long at = last + (slot - carry - before) * (long long)bt;
  if (at < of.R) return {kRest, (int)at, of.R};
  return {kNoRun, 0, 0};
}

// Zeros for the rows m0 .. m0 + rows - 1 of the columns in no run: chunk t.first, t.first + t.end, ... of 32 columns.  By the whole block.  (There is such a
// slot whenever there is such a column, see run_slots.)
template <typename T>
__device__ inline void clear_scattered(const Runs& of, const RunTile& t, T* C, long long ldc, int m0, int rows, RunSearch& s) {
  for (long long c0 = t.first * 32ll; c0 < of.R; c0 += t.end * 32ll) {
    if (threadIdx.x < 32) s.part[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < of.runs; i += blockDim.x)
      for (int n = max(of.begin(i), (int)c0); n < of.end(i) && n < c0 + 32; ++n) s.part[n - c0] = 1;
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * rows; i += blockDim.x) {
      const int n = i / rows, m = i % rows;
      if (c0 + n < of.R && !s.part[n]) C[(c0 + n) * ldc + m0 + m] = T(0.f);
    }
    __syncthreads();
  }
}

// tiles that R columns in `runs` runs can make, with the rest before and behind
__host__ __device__ inline long long run_slots(long long R, long long runs, int bt) {
  const long long cut = runs + 2 < R ? runs + 2 : R;
  return R / bt + cut;
}

}  // namespace
}  // namespace nb200
