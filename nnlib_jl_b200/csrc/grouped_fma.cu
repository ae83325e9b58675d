// Products of ragged groups of columns on the CUDA cores, exact fp32 in ascending k, any element type, size and stride.
//
//   grouped_fma_kernel   C[:, i] = A_g X[:, columns[i]] for the columns i of run g, and, for low-rank pairs, + B_a T[:, i]
//   grouped_grad_kernel  A_a = sum over the columns i of the runs of matrix a of C[:, i] X[:, columns[i]]^T
//
// Tiles and their shared-memory stages are gemm_fma.cu's: 256 threads, BT x BT, k in steps of 16, two stages.  A block's slot
// number is turned into (run, first column) by counting the tiles of all runs, since their sizes are on the device only; slots
// that no run needs end at once.  FMA bound: BT = 128 reads four 16-byte words of shared memory for 64 multiply-adds.
#include <algorithm>

#include "common.cuh"
#include "grouped_runs.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

// acc[i][j] += Q[k][i] * P[k][j] for a stage of BT + 4 wide rows
template <int BT>
struct Tile {
  static constexpr int KG = 16;
  static constexpr int R = BT / 16, G = R < 4 ? R : 4, LD = BT + 4, NL = BT * KG / 256;
  float acc[R][R];                           // [column side][row side]
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j) acc[i][j] = 0.f;
  }
  __device__ __forceinline__ void step(const float* p, const float* q, int tx, int ty) {
    float am[R], bn[R];
#pragma unroll
    for (int r = 0; r < R; r += G) {
      if constexpr (G == 4) {
        const float4 va = *reinterpret_cast<const float4*>(p + tx * 4 + r * 16);
        const float4 vb = *reinterpret_cast<const float4*>(q + ty * 4 + r * 16);
        am[r] = va.x; am[r + 1] = va.y; am[r + 2] = va.z; am[r + 3] = va.w;
        bn[r] = vb.x; bn[r + 1] = vb.y; bn[r + 2] = vb.z; bn[r + 3] = vb.w;
      } else {
        const float2 va = *reinterpret_cast<const float2*>(p + tx * 2);
        const float2 vb = *reinterpret_cast<const float2*>(q + ty * 2);
        am[0] = va.x; am[1] = va.y;
        bn[0] = vb.x; bn[1] = vb.y;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j) acc[i][j] = fmaf(am[j], bn[i], acc[i][j]);
  }
  static __device__ __forceinline__ int place(int t, int i) { return t * G + (i / G) * 16 * G + i % G; }
};

template <int BT>
struct Stages {
  float p[2][Tile<BT>::KG][Tile<BT>::LD], q[2][Tile<BT>::KG][Tile<BT>::LD];
};

// One contraction of K terms: P(k, row) and Q(k, column) give the elements (0 where there is none); `pk`: P's neighbours in
// memory are along k
template <int BT, typename FP, typename FQ>
__device__ __forceinline__ void contract(Tile<BT>& t, Stages<BT>& s, int K, bool pk, bool qk, FP P, FQ Q) {
  constexpr int NL = Tile<BT>::NL, KG = Tile<BT>::KG;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float rp[NL], rq[NL];
  auto at = [&](int e, bool along, int& k, int& r) {
    const int c = e * 256 + threadIdx.x;
    if (along) { k = c % KG; r = c / KG; } else { r = c % BT; k = c / BT; }
  };
  auto fetch = [&](int k0) {
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      int k, r;
      at(e, pk, k, r);
      rp[e] = k0 + k < K ? P(k0 + k, r) : 0.f;
      at(e, qk, k, r);
      rq[e] = k0 + k < K ? Q(k0 + k, r) : 0.f;
    }
  };
  auto stage = [&](int b) {
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      int k, r;
      at(e, pk, k, r);
      s.p[b][k][r] = rp[e];
      at(e, qk, k, r);
      s.q[b][k][r] = rq[e];
    }
  };
  if (K <= 0) return;
  fetch(0);
  __syncthreads();                           // (an earlier contraction's last stage has been read)
  stage(0);
  __syncthreads();
  for (int k0 = 0, b = 0; k0 < K; k0 += KG, b ^= 1) {
    const bool more = k0 + KG < K;
    if (more) fetch(k0 + KG);
    const int kn = min(KG, K - k0);         // the padding is not multiplied: 0 * Inf would be a NaN
    if (kn == KG) {
#pragma unroll
      for (int k = 0; k < KG; ++k) t.step(s.p[b][k], s.q[b][k], tx, ty);
    } else {
      for (int k = 0; k < kn; ++k) t.step(s.p[b][k], s.q[b][k], tx, ty);
    }
    if (more) stage(b ^ 1);
    __syncthreads();
  }
}

template <typename T, typename TC, int BT>
__global__ void __launch_bounds__(256) grouped_fma_kernel(const GroupedArgs g) {
  __shared__ __align__(16) Stages<BT> st;
  __shared__ RunSearch search;
  __shared__ int cols[BT];
  const RunTile run = find_run(Runs{g.offsets, g.run_len, g.G, g.R}, g.zero_rest, BT, blockIdx.x, search);
  if (run.run == kNoRun) return;
  const int m0 = blockIdx.y * BT, n0 = run.first, nn = min(BT, run.end - n0);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int mat = run.run < 0 ? -1 : (g.ids ? g.ids[run.run] : run.run);
  const bool have = mat >= 0 && mat < g.mats;
  for (int i = threadIdx.x; i < BT; i += 256) {
    int c = -1;
    if (have && i < nn) {
      c = g.columns ? g.columns[n0 + i] : n0 + i;
      if (c < 0 || c >= g.N) c = -1;
    }
    cols[i] = c;
  }
  __syncthreads();
  Tile<BT> t;
  t.clear();
  const T* X = reinterpret_cast<const T*>(g.X);
  if (have) {
    const T* A = reinterpret_cast<const T*>(g.A) + (long long)mat * g.strideA;
    contract<BT>(t, st, g.K, g.transA != 0, true,
                 [&](int k, int r) { return m0 + r < g.M ? Elem<T>::to_f(g.transA ? A[(long long)(m0 + r) * g.lda + k] : A[(long long)k * g.lda + m0 + r]) : 0.f; },
                 [&](int k, int r) { return cols[r] >= 0 ? Elem<T>::to_f(X[(long long)cols[r] * g.ldx + k]) : 0.f; });
  }
  const float scale = !have ? 0.f : (g.scale ? g.scale[mat] : g.scale0);
  if (scale != 1.f) {
#pragma unroll
    for (int i = 0; i < Tile<BT>::R; ++i)
#pragma unroll
      for (int j = 0; j < Tile<BT>::R; ++j) t.acc[i][j] *= scale;
  }
  if (g.low.r > 0) {
    // the runs of pairs that have columns here, one after the other; columns of other runs take no part
    const Runs of{g.low.offsets, g.low.run_len, g.low.runs, g.R};
    const float* low = reinterpret_cast<const float*>(g.low.T);
    for (int b = 0; b < g.low.runs; ++b) {
      const int lo = max(of.begin(b), n0), hi = min(of.end(b), n0 + nn), id = g.low.ids[b];
      if (lo >= hi || id < 0 || id >= g.low.n) continue;
      const T* B = reinterpret_cast<const T*>(g.low.B) + (long long)id * g.low.strideB;
      Tile<BT> u;
      u.clear();
      contract<BT>(u, st, g.low.r, g.low.transB != 0, true,
                   [&](int k, int r) { return m0 + r < g.M ? Elem<T>::to_f(g.low.transB ? B[(long long)(m0 + r) * g.low.ldb + k] : B[(long long)k * g.low.ldb + m0 + r]) : 0.f; },
                   [&](int k, int r) { return n0 + r >= lo && n0 + r < hi ? low[(long long)(n0 + r) * g.low.ldt + k] : 0.f; });
#pragma unroll
      for (int i = 0; i < Tile<BT>::R; ++i) {
        const int n = n0 + Tile<BT>::place(ty, i);
        if (n < lo || n >= hi) continue;     // (0 * Inf of another pair's matrix)
#pragma unroll
        for (int j = 0; j < Tile<BT>::R; ++j) t.acc[i][j] += u.acc[i][j];
      }
    }
  }
  TC* C = reinterpret_cast<TC*>(g.C);
#pragma unroll
  for (int i = 0; i < Tile<BT>::R; ++i) {
    const int c = Tile<BT>::place(ty, i);
    if (c >= nn) continue;
    const bool zero = cols[c] < 0;           // (a padding column's 0 times an infinity of A)
#pragma unroll
    for (int j = 0; j < Tile<BT>::R; ++j) {
      const int m = m0 + Tile<BT>::place(tx, j);
      if (m < g.M) C[(long long)(n0 + c) * g.ldc + m] = Elem<TC>::from_f(zero ? 0.f : t.acc[i][j]);
    }
  }
}

// blockIdx: (column tile of A, row tile of A, matrix).  Rows of A are C's, columns X's.
template <typename TC, typename TX, typename TA, int BT>
__global__ void __launch_bounds__(256) grouped_grad_kernel(const GroupedGradArgs g) {
  __shared__ __align__(16) Stages<BT> st;
  const int k0 = blockIdx.x * BT, m0 = blockIdx.y * BT, a = blockIdx.z;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const TC* C = reinterpret_cast<const TC*>(g.C);
  const TX* X = reinterpret_cast<const TX*>(g.X);
  const Runs of{g.offsets, g.run_len, g.G, g.R};
  Tile<BT> t;
  t.clear();
  for (int b = g.ids ? 0 : a; b < (g.ids ? g.G : min(a + 1, g.G)); ++b) {
    if (g.ids && g.ids[b] != a) continue;
    const int lo = of.begin(b), n = of.end(b) - lo;
    contract<BT>(t, st, n, false, false,
                 [&](int i, int r) {
                   if (m0 + r >= g.M) return 0.f;
                   if (g.columns && (unsigned)g.columns[lo + i] >= (unsigned)g.N) return 0.f;
                   return Elem<TC>::to_f(C[(long long)(lo + i) * g.ldc + m0 + r]);
                 },
                 [&](int i, int r) {
                   if (k0 + r >= g.K) return 0.f;
                   const int c = g.columns ? g.columns[lo + i] : lo + i;
                   return (unsigned)c < (unsigned)g.N ? Elem<TX>::to_f(X[(long long)c * g.ldx + k0 + r]) : 0.f;
                 });
  }
  TA* A = reinterpret_cast<TA*>(g.A) + (long long)a * g.strideA;
#pragma unroll
  for (int i = 0; i < Tile<BT>::R; ++i) {
    const int k = k0 + Tile<BT>::place(ty, i);
    if (k >= g.K) continue;
#pragma unroll
    for (int j = 0; j < Tile<BT>::R; ++j) {
      const int m = m0 + Tile<BT>::place(tx, j);
      if (m < g.M) A[g.transA ? (long long)m * g.lda + k : (long long)k * g.lda + m] = Elem<TA>::from_f(t.acc[i][j]);
    }
  }
}

template <typename T, typename TC, int BT>
cudaError_t launch(const GroupedArgs& g, cudaStream_t st) {
  const long long slots = run_slots(g.R, g.G, BT), rows = (g.M + BT - 1) / BT;
  if (slots > 0x7fffffffLL || rows > 65535) return cudaErrorInvalidConfiguration;
  grouped_fma_kernel<T, TC, BT><<<dim3((unsigned)slots, (unsigned)rows), 256, 0, st>>>(g);
  count_launch();
  return cudaGetLastError();
}
// The largest tile that is not mostly padding for runs of the average length and still gives most SMs a block: a tile of 32 reads twice as
// much shared memory for its products as one of 64 (333 x 200 by 1200 columns in 5 runs: 20 us in tiles of 32, 17 in tiles of 64).
template <typename T, typename TC>
cudaError_t launch_of(const GroupedArgs& g, cudaStream_t st) {
  if (g.M < 1 || g.R < 1) return cudaSuccess;
  const long long each = g.R / std::max(1, g.G);
  auto blocks = [&](long long bt) { return (g.R / bt + 1) * ((g.M + bt - 1) / bt); };
  if (each > 64 && g.M > 64 && blocks(128) >= 148) return launch<T, TC, 128>(g, st);
  if (each > 32 && g.M > 32 && blocks(64) >= 100) return launch<T, TC, 64>(g, st);
  return launch<T, TC, 32>(g, st);
}

template <typename TC, typename TX, typename TA, int BT>
cudaError_t launch_grad(const GroupedGradArgs& g, cudaStream_t st) {
  const long long rows = (g.M + BT - 1) / BT;
  if (rows > 65535 || g.mats > 65535) return cudaErrorInvalidConfiguration;
  grouped_grad_kernel<TC, TX, TA, BT><<<dim3((unsigned)((g.K + BT - 1) / BT), (unsigned)rows, (unsigned)g.mats), 256, 0, st>>>(g);
  count_launch();
  return cudaGetLastError();
}
// (there the sums are the runs', which a tile of 64 walks as long as one of 32: 25 us and 40)
template <typename TC, typename TX, typename TA>
cudaError_t launch_grad_of(const GroupedGradArgs& g, cudaStream_t st) {
  if (g.M < 1 || g.K < 1 || g.mats < 1) return cudaSuccess;
  auto blocks = [&](long long bt) { return ((g.K + bt - 1) / bt) * ((g.M + bt - 1) / bt) * g.mats; };
  if (g.M > 64 && g.K > 64 && blocks(128) >= 148) return launch_grad<TC, TX, TA, 128>(g, st);
  if (g.M > 32 && g.K > 32 && blocks(64) >= 148) return launch_grad<TC, TX, TA, 64>(g, st);
  return launch_grad<TC, TX, TA, 32>(g, st);
}

}  // namespace

// low: C is Float32, whatever A and X are
cudaError_t grouped_fma(const GroupedArgs& g, int dtype, bool f32_out, cudaStream_t st) {
  switch (dtype) {
    case NNLIB_B200_F16:  return f32_out ? launch_of<__half, float>(g, st) : launch_of<__half, __half>(g, st);
    case NNLIB_B200_BF16: return f32_out ? launch_of<__nv_bfloat16, float>(g, st) : launch_of<__nv_bfloat16, __nv_bfloat16>(g, st);
    default:              return launch_of<float, float>(g, st);
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
