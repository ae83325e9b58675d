// RMS norm of every query / key head and the rotation of its features by position in one pass, and the pullback.
//
//   r = 1 / sqrt(mean x^2 + eps),  n = x r g,  y = R n           (R turns feature pairs by position * frequency)
//   u = R^T dy,  w = u g,  dx = r (w - x r^2 mean(w x)),  dg = sum over tokens and heads of u x r
//
// Nothing is used twice but the angles, so HBM is the bound: x in and y out (pullback: x and dy in, dx out).  A group of
// `lanes` threads owns the row of one head, each lane V feature pairs (two 16-byte loads where the pairs' layout allows),
// so a row's sum takes log2(lanes) shuffles and a pair's two features never leave their thread.  A block takes TOK tokens;
// its angles (Float64 until they are reduced to one turn: a Float32 product of a position near 10^6 and a frequency would
// be off by 0.06) are worked out once, by all threads, and every group keeps those of its token in registers while it
// walks over that token's heads.  Queries and keys are two ranges of blocks of one launch.
// The weights' gradient: a thread's pairs are the same in every row it meets, so it sums in registers; the block adds its
// groups in a fixed order and leaves one row of partial sums in the workspace, norm_rope_reduce_kernel adds those in order.
#include <algorithm>

#include "common.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr int kNrThreads = 256;
constexpr int kNrMaxPairs = 128;      // d <= 256
constexpr int kNrMaxTok = 8;

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<2> { using type = unsigned short; };

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  using R = typename RawVec<V * sizeof(T)>::type;
  const R raw = __ldcs(reinterpret_cast<const R*>(p));
  T t[V];
  memcpy(t, &raw, sizeof(raw));
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = Elem<T>::to_f(t[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  using R = typename RawVec<V * sizeof(T)>::type;
  T t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = Elem<T>::from_f(in[i]);
  R raw;
  memcpy(&raw, t, sizeof(raw));
  *reinterpret_cast<R*>(p) = raw;
}

// the first feature of each of the two vectors of slot j (V pairs)
template <int V, bool INTER>
__device__ __forceinline__ void slot_features(const NormRopeArgs& a, int j, int& f0, int& f1) {
  if (INTER) {
    f0 = 2 * V * j;
    f1 = f0 + V;
  } else if (V * j < a.rot / 2) {
    f0 = V * j;
    f1 = f0 + a.rot / 2;
  } else {
    f0 = a.rot / 2 + V * j;            // rot + (V j - rot / 2)
    f1 = f0 + (a.d - a.rot) / 2;
  }
}

// NS: slots of a lane (1 with vectors; single pairs of a wide head are dealt out four to a lane)
template <typename T, int V, int NS, bool INTER, bool BWD>
__global__ void __launch_bounds__(kNrThreads) norm_rope_kernel(const NormRopeArgs a) {
  __shared__ float2 sm_turn[kNrMaxTok * kNrMaxPairs];
  const int pairs = a.d / 2, lanes = a.lanes, groups = kNrThreads / lanes, per_tok = groups / a.tok;
  const int tid = threadIdx.x, lane = tid % lanes, group = tid / lanes, tok = group / per_tok;
  const bool second = (int)blockIdx.x >= a.blocks_q;
  const NormRopeSide& s = a.side[second ? 1 : 0];
  const int bid = second ? blockIdx.x - a.blocks_q : blockIdx.x, nblk = second ? gridDim.x - a.blocks_q : a.blocks_q;
  const float inv_d = 1.f / (float)a.d;

  float gw[NS][2 * V], acc[NS][2 * V];
  int f0[NS], f1[NS];
  bool on[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int j = lane + n * lanes;
    on[n] = j * V < pairs;
    slot_features<V, INTER>(a, on[n] ? j : 0, f0[n], f1[n]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      gw[n][e] = load_bias(s.g, f0[n] + e, a.wdtype);
      gw[n][V + e] = load_bias(s.g, f1[n] + e, a.wdtype);
    }
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) acc[n][e] = 0.f;
  }

  for (long long tile = bid; tile * a.tok < a.tokens; tile += nblk) {
    const long long t0 = tile * a.tok;
    __syncthreads();                                     // the last tile's angles have been read
    for (int idx = tid; idx < a.tok * pairs; idx += kNrThreads) {
      const int tk = idx / pairs, p = idx - tk * pairs;
      float2 v = make_float2(1.f, 0.f);
      if (t0 + tk < a.tokens && 2 * p < a.rot) {
        const long long t = t0 + tk, b = t / a.L, l = t - b * a.L;
        const long long pos = a.positions ? (long long)a.positions[l * a.pos_sl + b * a.pos_sb]
                                          : l + (a.start ? (long long)a.start[b] : a.start0);
        const double turns = (double)pos * a.freqs[p] * 0.15915494309189533577;   // 1 / (2 pi)
        float sn, cs;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
        v = make_float2(cs, sn);
      }
      sm_turn[idx] = v;
    }
    __syncthreads();
    const long long t = t0 + tok;
    const bool token = t < a.tokens;
    const long long b = token ? t / a.L : 0, l = token ? t - b * a.L : 0;
    const T* xrow = reinterpret_cast<const T*>(s.x) + l * s.sl + b * s.sb;
    const T* dyrow = reinterpret_cast<const T*>(s.dy) + (BWD ? l * s.dsl + b * s.dsb : 0);
    T* orow = reinterpret_cast<T*>(s.out) + (token ? t : 0) * (long long)s.heads * a.d;
    float cs[NS][V], sn[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // pairs in the order of the registers: slot j holds pairs V j .. V j + V - 1
        const float2 v = sm_turn[tok * pairs + (on[n] ? (lane + n * lanes) * V + e : 0)];
        cs[n][e] = v.x;
        sn[n][e] = v.y;
      }
    // (the loop's length is the block's, so that a warp's shuffles find all of its lanes)
    for (int h0 = 0; h0 < s.heads; h0 += per_tok) {
      const int h = h0 + group - tok * per_tok;
      const bool live = token && h < s.heads;
      float x[NS][2 * V], u[NS][2 * V], sum = 0.f, dot = 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        if (live && on[n]) {
          load_vec<T, V>(xrow + (long long)h * a.d + f0[n], x[n]);
          load_vec<T, V>(xrow + (long long)h * a.d + f1[n], x[n] + V);
          if (BWD) {
            load_vec<T, V>(dyrow + (long long)h * a.d + f0[n], u[n]);
            load_vec<T, V>(dyrow + (long long)h * a.d + f1[n], u[n] + V);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) x[n][e] = u[n][e] = 0.f;
        }
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) sum = fmaf(x[n][e], x[n][e], sum);
      if (BWD) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
            const float da = u[n][ia], db = u[n][ib];
            u[n][ia] = fmaf(da, cs[n][e], db * sn[n][e]);
            u[n][ib] = fmaf(db, cs[n][e], -da * sn[n][e]);
          }
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) dot = fmaf(u[n][e] * gw[n][e], x[n][e], dot);
      }
      for (int off = lanes >> 1; off > 0; off >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (BWD) dot += __shfl_xor_sync(0xffffffffu, dot, off);
      }
      const float r = 1.f / sqrtf(fmaf(sum, inv_d, a.eps));
      const float back = BWD ? dot * inv_d * r * r : 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        if (BWD) {
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) {
            acc[n][e] = fmaf(u[n][e], x[n][e] * r, acc[n][e]);
            x[n][e] = r * fmaf(-x[n][e], back, u[n][e] * gw[n][e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) x[n][e] = x[n][e] * r * gw[n][e];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
            const float na = x[n][ia], nb = x[n][ib];
            x[n][ia] = fmaf(na, cs[n][e], -nb * sn[n][e]);
            x[n][ib] = fmaf(na, sn[n][e], nb * cs[n][e]);
          }
        }
        if (live && on[n]) {
          store_vec<T, V>(orow + (long long)h * a.d + f0[n], x[n]);
          store_vec<T, V>(orow + (long long)h * a.d + f1[n], x[n] + V);
        }
      }
    }
  }

  if (BWD) {
    // the block's sums: groups of a warp by shuffles, then the warps in order
    __syncthreads();
    float* sm = reinterpret_cast<float*>(sm_turn);       // 8 warps x 256 features
    static_assert(sizeof(sm_turn) >= kNrThreads / 32 * 2 * kNrMaxPairs * sizeof(float), "room for a row per warp");
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        float v = acc[n][e];
        for (int off = lanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if ((tid & 31) < lanes && on[n]) sm[(tid >> 5) * a.d + (e < V ? f0[n] + e : f1[n] + e - V)] = v;
      }
    __syncthreads();
    for (int f = tid; f < a.d; f += kNrThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kNrThreads / 32; ++w) v += sm[w * a.d + f];
      a.ws[(long long)blockIdx.x * a.d + f] = v;
    }
  }
}

// one block per 32 features and side: 32 rows of partial sums side by side, each thread its own in order
__global__ void __launch_bounds__(1024) norm_rope_reduce_kernel(const NormRopeArgs a, const int blocks) {
  __shared__ float sm[32][33];
  const int side = blockIdx.y, f = blockIdx.x * 32 + threadIdx.x;
  const int lo = side ? a.blocks_q : 0, hi = side ? blocks : a.blocks_q;
  float v = 0.f;
  if (f < a.d)
    for (int r = lo + threadIdx.y; r < hi; r += 32) v += a.ws[(long long)r * a.d + f];
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && f < a.d && a.side[side].dg) {
    v = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) v += sm[r][threadIdx.x];
    if (a.wdtype == NNLIB_B200_F16) reinterpret_cast<__half*>(a.side[side].dg)[f] = Elem<__half>::from_f(v);
    else if (a.wdtype == NNLIB_B200_BF16) reinterpret_cast<__nv_bfloat16*>(a.side[side].dg)[f] = Elem<__nv_bfloat16>::from_f(v);
    else reinterpret_cast<float*>(a.side[side].dg)[f] = v;
  }
}

// pairs of a vector: as many as fit 16 bytes, fewer where the layout of the pairs, a pointer or a stride asks for it
int vector_pairs(const NormRopeArgs& a, int esize, bool bwd) {
  for (int v = 16 / esize; v >= 4; v >>= 1) {
    bool ok = a.interleaved ? a.d % (2 * v) == 0 : (a.rot / 2) % v == 0 && ((a.d - a.rot) / 2) % v == 0;
    const long long bytes = (long long)v * esize;
    for (int i = 0; i < 2 && ok; ++i) {
      const NormRopeSide& s = a.side[i];
      if (!s.heads) continue;
      ok = (s.sl * esize) % bytes == 0 && (s.sb * esize) % bytes == 0 && (a.d * esize) % bytes == 0 &&
           reinterpret_cast<uintptr_t>(s.x) % bytes == 0 && reinterpret_cast<uintptr_t>(s.out) % bytes == 0;
      if (ok && bwd)
        ok = (s.dsl * esize) % bytes == 0 && (s.dsb * esize) % bytes == 0 && reinterpret_cast<uintptr_t>(s.dy) % bytes == 0;
    }
    if (ok) return v;
  }
  return 1;
}

int pow2_up(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

template <typename T, int V, int NS, bool BWD>
void launch(const NormRopeArgs& a, int blocks, cudaStream_t st) {
  if (a.interleaved) norm_rope_kernel<T, V, NS, true, BWD><<<blocks, kNrThreads, 0, st>>>(a);
  else norm_rope_kernel<T, V, NS, false, BWD><<<blocks, kNrThreads, 0, st>>>(a);
}

template <typename T, bool BWD>
void launch_v(const NormRopeArgs& a, int v, int blocks, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (v == 8) return launch<T, 8, 1, BWD>(a, blocks, st);
  }
  if (v == 4) return launch<T, 4, 1, BWD>(a, blocks, st);
  launch<T, 1, 4, BWD>(a, blocks, st);
}

// lanes of a row, tokens of a block and the blocks of both sides; returns their number
int plan(NormRopeArgs& a, int v, bool bwd) {
  const int pairs = a.d / 2, slots = (pairs + v - 1) / v;
  a.lanes = std::min(32, pow2_up(slots));
  const int groups = kNrThreads / a.lanes;
  const int heads = std::max(a.side[0].heads, a.side[1].heads);
  a.tok = 1;
  // four heads to a group where there are tokens enough to fill the GPU with it, else all of a token's heads at once
  while (a.tok * 2 <= std::min(groups, kNrMaxTok) && groups / (a.tok * 2) * 4 >= heads &&
         a.tokens / (a.tok * 2) >= 2 * 148) a.tok *= 2;
  const long long tiles = (a.tokens + a.tok - 1) / a.tok;
  const int hq = a.side[0].heads, hk = a.side[1].heads;
  const long long most = bwd ? 148 * 4 : 0x3fffffff;           // the pullback's blocks stay, for few partial sums
  long long nq = hq ? tiles : 0, nk = hk ? tiles : 0;
  if (nq + nk > most) {
    const long long share = hq && hk ? std::max<long long>(1, most * hq / (hq + hk)) : most;
    nq = hq ? std::min(nq, share) : 0;
    nk = hk ? std::min(nk, std::max<long long>(1, most - nq)) : 0;
  }
  a.blocks_q = (int)nq;
  return (int)(nq + nk);
}

}  // namespace

size_t norm_rope_workspace_bytes(NormRopeArgs a, int esize) {
  if (a.tokens == 0) return 0;
  return sizeof(float) * (size_t)plan(a, vector_pairs(a, esize, true), true) * a.d;
}

cudaError_t norm_rope(NormRopeArgs a, int dtype, bool bwd, cudaStream_t st) {
  const int v = vector_pairs(a, dtype == NNLIB_B200_F32 ? 4 : 2, bwd);
  const int blocks = a.tokens ? plan(a, v, bwd) : 0;
  if (blocks) {
    if (bwd) {
      if (dtype == NNLIB_B200_F16) launch_v<__half, true>(a, v, blocks, st);
      else if (dtype == NNLIB_B200_BF16) launch_v<__nv_bfloat16, true>(a, v, blocks, st);
      else launch_v<float, true>(a, v, blocks, st);
    } else {
      if (dtype == NNLIB_B200_F16) launch_v<__half, false>(a, v, blocks, st);
      else if (dtype == NNLIB_B200_BF16) launch_v<__nv_bfloat16, false>(a, v, blocks, st);
      else launch_v<float, false>(a, v, blocks, st);
    }
    count_launch();
  } else {
    a.blocks_q = 0;
  }
  if (bwd) {
    norm_rope_reduce_kernel<<<dim3((a.d + 31) / 32, 2), dim3(32, 32), 0, st>>>(a, blocks);
    count_launch();
  }
  return cudaGetLastError();
}

}  // namespace nb200
