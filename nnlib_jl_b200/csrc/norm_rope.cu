// RMS norm of every query / key head and the rotation of its features by position in one pass, and the pullback.
//
//   r = 1 / sqrt(mean x^2 + eps),  n = x r g,  y = R n           (R turns feature pairs by position * frequency)
//   u = R^T dy,  w = u g,  dx = r (w - x r^2 mean(w x)),  dg = sum over tokens and heads of u x r
//
// Nothing is used twice but the angles, so HBM is the bound (x in and y out; pullback: x and dy in, dx out) and what counts is
// rows in flight.  A group of `lanes` threads owns the row of one head, each lane V feature pairs (two 16-byte loads where
// the pairs' layout allows), so a row's sum takes a few shuffles and a pair's two features never leave their thread.  A warp
// holds as many groups as fit (six of five lanes for a head of 80 features) and works by itself: it takes a token, or some of
// a token's heads where tokens are few, works out its angles, and walks over the heads, the next rows, then the next token's,
// always under way.  Queries and keys are two ranges of blocks of one launch.
// bf16, 32768 tokens, heads of 128: 32 + 8 heads 135 us (5.0 TB/s), pullback 273 (3.7; Float32 weights, whose
// gradients ask for better sines, 275); 32 + 32 heads 196 (5.5) and 381 (4.2; 387);
// Float32, 16384 tokens, 32 + 8 heads 122 (5.5) and 168 (6.0): what bounds the 16-bit pullback is the number of rows under
// way, 64 to an SM at 128 registers a thread, and the issue slots that a row takes however many bytes it has.  Float16, 6000
// tokens, 8 + 8 heads of 80: 13.5 and 29.4 (2.3 and 1.6 TB/s): four or five tokens to a warp, each a chain of angles, shared
// memory and rows, and eight heads are six rows and two for its six groups.
// The weights' gradient: a thread's pairs are the same in every row it meets, so it sums in registers; the block adds its
// groups in a fixed order and leaves one row of partial sums in the workspace, norm_rope_reduce_kernel adds those in order.
#include <algorithm>

#include "common.cuh"
#include "launchers.h"
#include "umma.cuh"

namespace nb200 {
namespace {

constexpr int kNrThreads = 128, kNrWarps = kNrThreads / 32, kNrMaxPairs = 128;   // d <= 256

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<2> { using type = unsigned short; };
template <typename T, int V>
using VecOf = typename RawVec<V * sizeof(T)>::type;

// Arithmetic is on two Float32 numbers at a time (half the instructions; without it the pullback is short of issue slots)
using ptx::pair_add;
using ptx::pair_fma;
using ptx::pair_mul;
using ptx::pair_of;
using ptx::pair_pack;
using ptx::pair_sum;
using ptx::pair_unpack;
typedef unsigned long long Two;
__device__ __forceinline__ Two swapped(Two v) {
  float lo, hi;
  pair_unpack(v, lo, hi);
  return pair_pack(hi, lo);
}

// the V elements of a vector, two by two
template <typename T, int V>
__device__ __forceinline__ void unpack(const VecOf<T, V>& raw, Two* out) {
  T t[V];
  memcpy(t, &raw, sizeof(raw));
#pragma unroll
  for (int i = 0; i < V / 2; ++i) out[i] = pair_pack(Elem<T>::to_f(t[2 * i]), Elem<T>::to_f(t[2 * i + 1]));
}
__device__ __forceinline__ uint32_t two16(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  uint32_t u;
  memcpy(&u, &v, 4);
  return u;
}
__device__ __forceinline__ uint32_t two16(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  uint32_t u;
  memcpy(&u, &v, 4);
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Two* in) {
  VecOf<T, V> raw;
  if constexpr (sizeof(T) == 4) {
    memcpy(&raw, in, sizeof(raw));
  } else {
    uint32_t t[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float lo, hi;
      pair_unpack(in[i], lo, hi);
      t[i] = two16(lo, hi, T());
    }
    memcpy(&raw, t, sizeof(raw));
  }
  *reinterpret_cast<VecOf<T, V>*>(p) = raw;
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

// the sum over a group's lanes (gl: this lane's place in it, first: the warp's lane that is its first)
__device__ __forceinline__ float group_sum(float v, int lanes, int gl, int first) {
  if ((lanes & (lanes - 1)) == 0) {
    for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  }
  for (int off = lanes > 16 ? 16 : (lanes > 8 ? 8 : (lanes > 4 ? 4 : 2)); off > 0; off >>= 1) {
    const float t = __shfl_down_sync(0xffffffffu, v, off);
    if (gl + off < lanes) v += t;
  }
  return __shfl_sync(0xffffffffu, v, first);
}

// NS: slots of a lane (1 with vectors; single pairs of a wide head are dealt out four to a lane)
template <typename T, int V, int NS, bool INTER, bool BWD>
__global__ void __launch_bounds__(kNrThreads, V == 1 ? 3 : (BWD && V == 8 ? 4 : 5)) norm_rope_kernel(const NormRopeArgs a) {
  using R = VecOf<T, V>;
  // Two numbers of a register pair: a feature pair (ADJ), or neighbours of one half of the head, the other half's behind
  constexpr bool ADJ = INTER || V == 1;
  constexpr int H2 = V / 2;
  const int lanes = a.lanes, per_warp = 32 / lanes, pairs = a.d / 2;
  const int wl = threadIdx.x & 31, warp = threadIdx.x >> 5, wg = wl / lanes, lane = wl - wg * lanes;
  const bool here = wg < per_warp;                       // lanes behind the last whole group keep their warp company
  const bool second = (int)blockIdx.x >= a.blocks_q;
  const NormRopeSide& s = a.side[second ? 1 : 0];
  const int bid = second ? blockIdx.x - a.blocks_q : blockIdx.x, nblk = second ? gridDim.x - a.blocks_q : a.blocks_q;
  const float inv_d = 1.f / (float)a.d;
  const bool whole = a.rot == a.d;                       // every feature is turned

  Two gw[NS][V], acc[NS][V];
  int f0[NS], f1[NS];
  bool on[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int j = lane + n * lanes;
    on[n] = here && j * V < pairs;
    slot_features<V, INTER>(a, on[n] ? j : 0, f0[n], f1[n]);
    float g[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      g[e] = load_bias(s.g, f0[n] + e, a.wdtype);
      g[V + e] = load_bias(s.g, f1[n] + e, a.wdtype);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      gw[n][e] = pair_pack(g[2 * e], g[2 * e + 1]);
      acc[n][e] = 0ull;
    }
  }

  // Frequencies in turns per position, the fraction as 64 bits: a position times that, whose overflow are whole turns, is the
  // angle to 2^-32 of a turn for frequencies up to 1 and positions below 2^23, to 2^-24 at 2^31, where the frequency's own last
  // bits count (a Float32 product near 10^6 would be off by 0.06, and Float64 arithmetic for every token and pair costs more
  // issue slots than the row)
  __shared__ unsigned long long sm_freq[kNrMaxPairs];
  __shared__ float2 sm_turn[kNrWarps][kNrMaxPairs];
  __shared__ float sm_one[kNrMaxPairs];                  // NaN for a frequency that is not finite
  for (int p = threadIdx.x; p < pairs; p += kNrThreads) {
    double t = 2 * p < a.rot ? a.freqs[p] * 0.15915494309189533577 : 0.0;   // 1 / (2 pi)
    sm_one[p] = t - t == 0.0 ? 1.f : __int_as_float(0x7fc00000);
    t -= floor(t);
    sm_freq[p] = (unsigned long long)(t * 18446744073709551616.0);
  }
  __syncthreads();

  // a unit: one token and s.chunk of its heads
  const unsigned chunks = (s.heads + s.chunk - 1) / s.chunk, units = (unsigned)a.tokens * chunks, step = nblk * kNrWarps;
  const T *xrow, *dyrow;
  T* orow;
  long long pos;
  int h_lo, h_hi;
  auto place = [&](unsigned u) {
    const unsigned t = u / chunks, c = u - t * chunks, b = t / (unsigned)a.L, l = t - b * a.L;
    h_lo = c * s.chunk;
    h_hi = min(s.heads, h_lo + s.chunk);
    xrow = reinterpret_cast<const T*>(s.x) + l * s.sl + b * s.sb;
    dyrow = BWD ? reinterpret_cast<const T*>(s.dy) + l * s.dsl + b * s.dsb : nullptr;
    orow = reinterpret_cast<T*>(s.out) + (long long)t * s.heads * a.d;
    pos = a.positions ? (long long)a.positions[l * a.pos_sl + b * a.pos_sb] : l + (a.start ? (long long)a.start[b] : a.start0);
  };
  R xr[NS][2], dr[NS][2];
  auto fetch = [&](int h) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (!(on[n] && h + wg < h_hi)) continue;
      const int at = (h + wg) * a.d;
      xr[n][0] = __ldcs(reinterpret_cast<const R*>(xrow + at + f0[n]));
      xr[n][1] = __ldcs(reinterpret_cast<const R*>(xrow + at + f1[n]));
      if (BWD) {
        dr[n][0] = __ldcs(reinterpret_cast<const R*>(dyrow + at + f0[n]));
        dr[n][1] = __ldcs(reinterpret_cast<const R*>(dyrow + at + f1[n]));
      }
    }
  };
  unsigned unit = bid * kNrWarps + warp;
  if (unit < units) {
    place(unit);
    fetch(h_lo);
  }
  while (unit < units) {
    // The token's angles, by all lanes.  Forward: the weights go into the factors, y_a = r (x_a ga cos - x_b gb sin),
    // y_b = r (x_a ga sin + x_b gb cos).
    __syncwarp();
    for (int p = wl; p < pairs; p += 32) {
      const float one = sm_one[p], turns = (float)(int)((sm_freq[p] * (unsigned long long)pos) >> 32) * 2.3283064365386963e-10f;
      float tc, ts;
      // (16-bit results: sine and cosine to 2^-21; not where the weights' gradients are Float32)
      if (sizeof(T) == 2 && !(BWD && a.wdtype == NNLIB_B200_F32)) __sincosf(6.283185307179586f * turns, &ts, &tc);
      else sincospif(2.f * turns, &ts, &tc);
      sm_turn[warp][p] = make_float2(tc * one, ts * one);
    }
    __syncwarp();
    Two f1c[NS][V], f2s[NS][V];      // ADJ: of the number itself and of its partner; else cos of both halves, sin (a: -, b: +)
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      float c[V], w[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 t = sm_turn[warp][on[n] ? (lane + n * lanes) * V + e : 0];
        c[e] = t.x;
        w[e] = BWD ? -t.y : t.y;     // the opposite angle
      }
      if constexpr (ADJ) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          f1c[n][e] = pair_of(c[e]);
          f2s[n][e] = pair_pack(-w[e], w[e]);
          if (!BWD) {
            f1c[n][e] = pair_mul(f1c[n][e], gw[n][e]);
            f2s[n][e] = pair_mul(f2s[n][e], swapped(gw[n][e]));
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < H2; ++e) {
          f1c[n][e] = f1c[n][H2 + e] = pair_pack(c[2 * e], c[2 * e + 1]);
          f2s[n][e] = pair_pack(-w[2 * e], -w[2 * e + 1]);
          f2s[n][H2 + e] = pair_pack(w[2 * e], w[2 * e + 1]);
          if (!BWD) {
            f1c[n][e] = pair_mul(f1c[n][e], gw[n][e]);
            f1c[n][H2 + e] = pair_mul(f1c[n][H2 + e], gw[n][H2 + e]);
            f2s[n][e] = pair_mul(f2s[n][e], gw[n][H2 + e]);
            f2s[n][H2 + e] = pair_mul(f2s[n][H2 + e], gw[n][e]);
          }
        }
      }
    }
    auto partner = [&](const Two (&v)[V], int e) { return ADJ ? swapped(v[e]) : v[e < H2 ? e + H2 : e - H2]; };
    // The rotation of slot n.  Features that are not turned meet no other: the sine of 0 would make NaN of an infinity there.
    // (plain: every feature is turned, or v holds none)
    auto turned = [&](const Two (&v)[V], int n, bool plain, Two (&t)[V]) {
      if (plain) {
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = pair_fma(v[e], f1c[n][e], pair_mul(partner(v, e), f2s[n][e]));
      } else {
        const int left = a.rot / 2 - (lane + n * lanes) * V;      // pairs of this slot that are turned
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const Two other = (ADJ ? e < left : left > 0) ? partner(v, e) : 0ull;
          t[e] = pair_fma(v[e], f1c[n][e], pair_mul(other, f2s[n][e]));
        }
      }
    };
    const int h_end = h_hi;
    T* const out = orow;
    for (int h = h_lo; h < h_end; h += per_warp) {       // (the same for all of a warp's lanes: they shuffle)
      const bool live = here && h + wg < h_end;
      Two x[NS][V], u[NS][V], sum2 = 0ull, dot2 = 0ull;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        if (live && on[n]) {
          if constexpr (V == 1) {
            T e[2];
            memcpy(&e[0], &xr[n][0], sizeof(T));
            memcpy(&e[1], &xr[n][1], sizeof(T));
            x[n][0] = pair_pack(Elem<T>::to_f(e[0]), Elem<T>::to_f(e[1]));
            if (BWD) {
              memcpy(&e[0], &dr[n][0], sizeof(T));
              memcpy(&e[1], &dr[n][1], sizeof(T));
              u[n][0] = pair_pack(Elem<T>::to_f(e[0]), Elem<T>::to_f(e[1]));
            }
          } else {
            unpack<T, V>(xr[n][0], x[n]);
            unpack<T, V>(xr[n][1], x[n] + H2);
            if (BWD) {
              unpack<T, V>(dr[n][0], u[n]);
              unpack<T, V>(dr[n][1], u[n] + H2);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) x[n][e] = u[n][e] = 0ull;
        }
      }
      if (h + per_warp < h_end) {
        fetch(h + per_warp);
      } else if (unit + step < units) {
        place(unit + step);
        fetch(h_lo);
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) sum2 = pair_fma(x[n][e], x[n][e], sum2);
      Two w[NS][V];
      if (BWD) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          Two t[V];
          turned(u[n], n, whole, t);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            u[n][e] = t[e];
            w[n][e] = pair_mul(t[e], gw[n][e]);
            dot2 = pair_fma(w[n][e], x[n][e], dot2);
          }
        }
      }
      const float sum = group_sum(pair_sum(sum2), lanes, lane, wl - lane);
      // (the approximation's error, two units in the last place, is little beside the sum's)
      // A group that has no row this time must add nothing to the weights' gradient: with eps = 0 its r would be infinite.
      const float r = rsqrtf(fmaf(sum, inv_d, live || !BWD ? a.eps : 1.f));
      const Two r2 = pair_of(r);
      Two back2 = 0ull;
      if (BWD) back2 = pair_of(-group_sum(pair_sum(dot2), lanes, lane, wl - lane) * inv_d * r * r);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        Two y[V];
        if (!BWD) turned(x[n], n, sum <= 3.402823466e38f, y);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (BWD) {
            const Two xs = pair_mul(x[n][e], r2);
            acc[n][e] = pair_fma(u[n][e], xs, acc[n][e]);
            y[e] = pair_fma(xs, back2, pair_mul(w[n][e], r2));
          } else {
            y[e] = pair_mul(r2, y[e]);
          }
        }
        if (live && on[n]) {
          T* const o = out + (h + wg) * a.d;
          if constexpr (V == 1) {
            float lo, hi;
            pair_unpack(y[0], lo, hi);
            o[f0[n]] = Elem<T>::from_f(lo);
            o[f1[n]] = Elem<T>::from_f(hi);
          } else {
            store_vec<T, V>(o + f0[n], y);
            store_vec<T, V>(o + f1[n], y + H2);
          }
        }
      }
    }
    unit += step;
  }

  if (BWD) {
    // the block's sums: its groups in order
    __shared__ float sm[BWD ? kNrThreads * 2 * V * NS : 1];   // groups x d: a lane holds at most 2 V NS features
    const int groups = kNrWarps * per_warp, group = warp * per_warp + wg;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (on[n]) {
          float lo, hi;
          pair_unpack(acc[n][e], lo, hi);
          // numbers 2e and 2e + 1 of the slot's two vectors
          sm[group * a.d + (2 * e < V ? f0[n] + 2 * e : f1[n] + 2 * e - V)] = lo;
          sm[group * a.d + (2 * e + 1 < V ? f0[n] + 2 * e + 1 : f1[n] + 2 * e + 1 - V)] = hi;
        }
    __syncthreads();
    for (int f = threadIdx.x; f < a.d; f += kNrThreads) {
      float v = 0.f;
      for (int w = 0; w < groups; ++w) v += sm[w * a.d + f];
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
  if (f < a.d) {
#pragma unroll 8
    for (int r = lo + threadIdx.y; r < hi; r += 32) v += a.ws[(long long)r * a.d + f];
  }
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

// lanes of a row, heads of a unit and the blocks of both sides; returns their number
int plan(NormRopeArgs& a, int v, bool bwd) {
  const int pairs = a.d / 2;
  a.lanes = std::min(32, (pairs + v - 1) / v);
  const int per_warp = 32 / a.lanes;
  const int fit = bwd && v == 8 ? 4 : 5;                       // blocks of an SM (the kernel's launch bound)
  const long long slots = 148 * fit * kNrWarps;
  long long n[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    NormRopeSide& s = a.side[i];
    if (!s.heads) continue;
    // a token's heads are cut up only where tokens alone leave warps without work
    const long long cut = std::max(1LL, std::min<long long>((s.heads + per_warp - 1) / per_warp, slots / std::max(a.tokens, 1LL)));
    s.chunk = (int)((s.heads + cut - 1) / cut);
    n[i] = (a.tokens * ((s.heads + s.chunk - 1) / s.chunk) + kNrWarps - 1) / kNrWarps;
  }
  // Blocks stay and take unit after unit; both sides get what their heads are worth.  A row of keys costs more than one of
  // queries where there are fewer of them to a token, and the pullback evens that out with twice the blocks that fit (bf16,
  // 32 and 8 heads of 128, 32768 tokens: 304 -> 276 us; 32 and 32 heads 383 and 387), if they have work for it.
  const long long most = 148LL * fit * (bwd && v == 8 && (n[0] + n[1]) / (148 * fit) >= 16 ? 2 : 1);
  if (n[0] + n[1] > most) {
    const int hq = a.side[0].heads, hk = a.side[1].heads;
    const long long share = hk == 0 ? most : hq == 0 ? 0 : std::max(1LL, std::min(most - 1, (most * hq + (hq + hk) / 2) / (hq + hk)));
    n[0] = std::min(n[0], share);
    n[1] = std::min(n[1], most - share);
  }
  a.blocks_q = (int)n[0];
  return (int)(n[0] + n[1]);
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
