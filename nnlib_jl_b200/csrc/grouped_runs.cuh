// Runs of columns whose ends are on the device: what a block does to find the tile that is its own.
#pragma once

#include <cuda_runtime.h>

namespace nb200 {
namespace {

constexpr int kRest = -1;                // a tile of columns in no run, before the first or behind the last
constexpr int kNoRun = -2;               // no tile at all

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

// Tile number `slot` when the columns before the first run (rest), of every run in turn and behind the last one (rest) are
// cut into tiles of bt columns.  Called by a whole block of whole warps.
__device__ inline RunTile find_run(const Runs& of, bool rest, int bt, int slot, RunSearch& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (threadIdx.x == 0) s.found = {kNoRun, 0, 0};
  int carry = 0;
  for (int i0 = -1; i0 <= of.runs; i0 += blockDim.x) {
    const int i = i0 + (int)threadIdx.x;
    int first = 0, end = 0;
    if (i == -1) { if (rest) end = of.runs > 0 ? of.at(0) : of.R; }
    else if (i < of.runs) { first = of.begin(i); end = of.end(i); }
    else if (i == of.runs && rest && of.runs > 0) { first = of.at(of.runs); end = of.R; }
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
    if (at >= 0 && at < own) s.found = {i < 0 || i >= of.runs ? kRest : i, first + at * bt, end};
    carry = all;
    __syncthreads();
    if (slot < carry) break;             // (the same for every thread)
  }
  return s.found;
}

// tiles that R columns in `runs` runs can make, with the rest before and behind
__host__ __device__ inline long long run_slots(long long R, long long runs, int bt) {
  const long long cut = runs + 2 < R ? runs + 2 : R;
  return R / bt + cut;
}

}  // namespace
}  // namespace nb200
