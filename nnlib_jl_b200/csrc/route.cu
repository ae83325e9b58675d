// The router of a layer of experts and the sum that ends it (include/nnlib_b200.h: nnlib_b200_route, nnlib_b200_combine).
//
// route: S_t = the k largest of l_t + b; w = softmax(l) over S_t or over all; then a stable counting sort of the chosen
// (token, expert) pairs by expert.  A warp takes a token: its G logits are order-preserving integers in registers, in falling order in
// each lane, and k times the largest head is taken (redux.sync gives a warp's largest; the first lane that has it has the lowest expert, since
// lanes hold neighbouring experts).  A block counts its tokens' choices; a second launch turns the counts of all blocks into each
// block's first number for each expert; a third gives every pair its number: a token picks an expert at most once, so the
// pair's place among its block's is the number of earlier tokens in the expert's bit mask.  Nothing depends on the order in
// which warps run.  Few tokens take one block and one launch.  What bounds it is instructions, 547 a token of 256 experts and 8 choices (32768 such
// tokens, bf16: 26 + 8 + 10 us).
//
// combine: HBM bound, 16 bytes a thread and column (8192 tokens of 2 columns of 4096, bf16: 42 us, 4.7 TB/s; the pullback of 4096 tokens of 6
// columns of 2048: 40 us, 5.4 TB/s).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "early.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
constexpr int kChooseWarps = 8;
constexpr int kMaxPerBlock = 256;        // tokens whose choices one block numbers: the masks of an expert are 8 words

// Larger floats are larger integers; -0 like +0; NaN below everything; 0 for what cannot be chosen.
__device__ __forceinline__ unsigned sortable(float x) {
  if (isnan(x)) return 1u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// What an expert is chosen by, unlike any other's: its logit, then the lower expert.  A 16-bit logit fits one word with the
// expert's number.
__device__ __forceinline__ unsigned packed_key(unsigned bits, unsigned infinity, int e) {
  const unsigned size = bits & 0x7fffu;
  unsigned k = (bits & 0x8000u) ? 0x8000u - size : 0x8000u + size;      // -0 like +0
  if (size > infinity) k = 0u;                                          // NaN
  return k << 16 | (0xffffu - (unsigned)e);
}
template <typename T> __device__ __forceinline__ unsigned raw_bits(T v) { return 0u; }
template <> __device__ __forceinline__ unsigned raw_bits(__half v) { return __half_as_ushort(v); }
template <> __device__ __forceinline__ unsigned raw_bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ unsigned long long wide_key(float x, int e) {
  return (unsigned long long)sortable(x) << 32 | (0xffffffffu - (unsigned)e);
}
// in falling order: Batcher's odd-even merge sort
template <int V, typename K>
__device__ __forceinline__ void sort_falling(K (&a)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2) {
#pragma unroll
    for (int k = p; k >= 1; k /= 2) {
#pragma unroll
      for (int i = 0; i + k < V; ++i) {
        const bool in = i >= k % p && ((i - k % p) / k) % 2 == 0 && i / (2 * p) == (i + k) / (2 * p);
        if (in) {
          const K lo = a[i] < a[i + k] ? a[i] : a[i + k], hi = a[i] < a[i + k] ? a[i + k] : a[i];
          a[i] = hi;
          a[i + k] = lo;
        }
      }
    }
  }
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// V neighbouring logits of a token for each lane; -Inf where there is no expert.  vec: as many as fit 16 bytes at a time
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* row, int G, int lane, bool vec, T (&x)[V]) {
  constexpr int W = V * sizeof(T) <= 16 ? V : 16 / sizeof(T);
  if (vec && lane * V + V <= G) {
#pragma unroll
    for (int v = 0; v < V; v += W) {
      const Pack<T, W> p = *reinterpret_cast<const Pack<T, W>*>(row + lane * V + v);
#pragma unroll
      for (int w = 0; w < W; ++w) x[v + w] = p.v[w];
    }
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    x[v] = e < G ? row[e] : Elem<T>::from_f(__int_as_float(0xff800000));
  }
}
// the exponential of a logit relative to the largest: the slow branch of the softmax for +Inf
__device__ __forceinline__ float share_of(float x, float mx) {
  if (mx == __int_as_float(0x7f800000)) return x == mx ? 1.f : (isnan(x) ? x : 0.f);
  return expf(x - mx);
}

template <typename T, int V, bool PACKED>
__device__ void choose_token(const RouteArgs& a, int t, int lane, int* count) {
  const bool live = !a.mask || a.mask[t];
  int mine = -1;                          // lane j: the j-th expert of the token
  float w = 0.f;
  if (live) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)t * a.stride;
    T x[V];
    load_logits<T, V>(row, a.G, lane, a.vec != 0, x);
    // every lane's experts in falling order: the warp's best is the best of their heads
    typename std::conditional<PACKED, unsigned, unsigned long long>::type key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if constexpr (PACKED) {
        key[v] = e < a.G ? packed_key(raw_bits(x[v]), std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u, e) : 0u;
      } else {
        const float f = Elem<T>::to_f(x[v]);
        key[v] = e < a.G ? wide_key(a.bias ? f + a.bias[e] : f, e) : 0ull;
      }
    }
    sort_falling<V>(key);
    for (int j = 0; j < a.k; ++j) {
      int e;
      bool win;
      if constexpr (PACKED) {
        const unsigned top = __reduce_max_sync(kFull, key[0]);
        e = (int)(0xffffu - (top & 0xffffu));
        win = key[0] == top;
      } else {
        const unsigned head = (unsigned)(key[0] >> 32), top = __reduce_max_sync(kFull, head);
        const int src = __ffs(__ballot_sync(kFull, head == top)) - 1;      // (lanes hold neighbouring experts)
        e = (int)(0xffffffffu - __shfl_sync(kFull, (unsigned)key[0], src));
        win = lane == src;
      }
      if (lane == j) mine = e;
      if (win) {
#pragma unroll
        for (int v = 0; v + 1 < V; ++v) key[v] = key[v + 1];
        key[V - 1] = 0;
      }
    }
    const float logit = lane < a.k ? Elem<T>::to_f(row[mine]) : 0.f;
    if (a.normalize) {
      // over the first lanes only: as many steps as k has bits
      float mx = lane < a.k ? logit : __int_as_float(0xff800000);
      for (int o = a.k_up / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
      const float part = lane < a.k ? share_of(logit, mx) : 0.f;
      float sum = part;
      for (int o = a.k_up / 2; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      w = part / sum;
    } else {
      float mx = Elem<T>::to_f(x[0]), part = 0.f;
#pragma unroll
      for (int v = 1; v < V; ++v) mx = fmaxf(mx, Elem<T>::to_f(x[v]));
      mx = warp_max(mx);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane * V + v < a.G) part += share_of(Elem<T>::to_f(x[v]), mx);
      w = share_of(logit, mx) / warp_sum(part);
    }
    if (count && lane < a.k) atomicAdd(&count[mine], 1);
  }
  if (lane < a.k) {
    const long long o = (long long)t * a.k + lane;
    a.experts[o] = mine;
    a.weights[o] = w;
  }
}

// exclusive sums of n values in shared memory by a block of 32 * W threads; returns the total
template <int W>
__device__ int block_scan(int* v, int n, int* part) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int carry = 0;
  for (int i0 = 0; i0 < n; i0 += 32 * W) {
    const int i = i0 + threadIdx.x;
    const int own = i < n ? v[i] : 0;
    int s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) part[warp] = s;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      if (q < warp) before += part[q];
      all += part[q];
    }
    if (i < n) v[i] = before + s - own;
    carry = all;
    __syncthreads();
  }
  return carry;
}

// Numbers of the pairs of tokens t0 .. t1 - 1; base[e]: the first number of expert e here; mask: 8 words for each expert
__device__ void number_pairs(const RouteArgs& a, int t0, int t1, const int* base, unsigned* mask) {
  const int n = (t1 - t0) * a.k;
  for (int i = threadIdx.x; i < a.G * (kMaxPerBlock / 32); i += blockDim.x) mask[i] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int e = a.experts[(long long)t0 * a.k + i], t = i / a.k;
    if (e >= 0) atomicOr(&mask[e * (kMaxPerBlock / 32) + (t >> 5)], 1u << (t & 31));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const long long o = (long long)t0 * a.k + i;
    const int e = a.experts[o], t = i / a.k;
    int at = -1;
    if (e >= 0) {
      const unsigned* m = mask + e * (kMaxPerBlock / 32);
      at = base[e] + __popc(m[t >> 5] & ((1u << (t & 31)) - 1u));
      for (int q = 0; q < (t >> 5); ++q) at += __popc(m[q]);
      a.columns[at] = t0 + t;
    }
    a.position[o] = at;
  }
}
__device__ void end_of_order(const RouteArgs& a, int total, long long i0, long long i1) {
  for (long long i = (i0 > total ? i0 : total) + threadIdx.x; i < i1; i += blockDim.x) a.columns[i] = -1;
}

// shared memory: G counts or bases, then the masks
template <typename T, int V, bool PACKED, bool ALONE, int W>
__global__ void __launch_bounds__(32 * W) route_choose_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  __shared__ int part[W];
  const int t0 = blockIdx.x * a.per_block, t1 = min(a.N, t0 + a.per_block);
  let_next();
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  for (int t = t0 + (threadIdx.x >> 5); t < t1; t += W) choose_token<T, V, PACKED>(a, t, threadIdx.x & 31, sm);
  __syncthreads();
  if constexpr (ALONE) {
    const int total = block_scan<W>(sm, a.G, part);
    for (int i = threadIdx.x; i < a.G; i += blockDim.x) a.offsets[i] = sm[i];
    if (threadIdx.x == 0) a.offsets[a.G] = total;
    number_pairs(a, t0, t1, sm, reinterpret_cast<unsigned*>(sm + a.G));
    end_of_order(a, total, 0, (long long)a.N * a.k);
  } else {
    for (int i = threadIdx.x; i < a.G; i += blockDim.x) a.ws[(long long)i * a.blocks + blockIdx.x] = sm[i];
  }
}

// counts of each expert, block by block, to the number of its pairs in earlier blocks; a warp an expert
__global__ void __launch_bounds__(256) route_scan_kernel(const RouteArgs a) {
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  let_next();
  wait_before();
  if (e >= a.G) return;
  int* c = a.ws + (long long)e * a.blocks;
  int carry = 0;
  for (int i0 = 0; i0 < a.blocks; i0 += 256) {             // eight neighbours a lane: all on their way at once
    int own[8], sum = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + lane * 8 + u;
      own[u] = i < a.blocks ? c[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += own[u];
    int s = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += u;
    }
    int before = carry + s - sum;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + lane * 8 + u;
      if (i < a.blocks) c[i] = before;
      before += own[u];
    }
    carry += __shfl_sync(kFull, s, 31);
  }
  if (lane == 0) a.ws[(long long)a.G * a.blocks + e] = carry;
}

__global__ void __launch_bounds__(256) route_number_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  __shared__ int part[8];
  wait_before();
  const int* totals = a.ws + (long long)a.G * a.blocks;
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) sm[i] = totals[i];
  __syncthreads();
  const int total = block_scan<8>(sm, a.G, part);
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.G; i += blockDim.x) a.offsets[i] = sm[i];
    if (threadIdx.x == 0) a.offsets[a.G] = total;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) sm[i] += a.ws[(long long)i * a.blocks + blockIdx.x];
  __syncthreads();
  const int t0 = blockIdx.x * a.per_block, t1 = min(a.N, t0 + a.per_block);
  number_pairs(a, t0, t1, sm, reinterpret_cast<unsigned*>(sm + a.G));
  end_of_order(a, total, (long long)t0 * a.k, (long long)t1 * a.k);
}

// dl = w (dw - sum w dw) at the chosen; or, not normalised, p (d - sum w dw) with d = dw at the chosen, 0 elsewhere
template <typename T, int V>
__global__ void __launch_bounds__(256) route_bwd_kernel(const RouteArgs a) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= a.N) return;
  int e = -1;
  float w = 0.f, dw = 0.f;
  if (lane < a.k) {
    const long long o = (long long)t * a.k + lane;
    e = a.experts[o];
    if (e >= 0) { w = a.weights[o]; dw = a.dweights[o]; }
  }
  const bool live = __any_sync(kFull, e >= 0);
  const float mean = warp_sum(w * dw);
  float d[V];
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = 0.f;
  const float mine = a.normalize ? w * (dw - mean) : dw;
  for (int j = 0; j < a.k; ++j) {
    const int at = __shfl_sync(kFull, e, j) - lane * V;
    const float val = __shfl_sync(kFull, mine, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v == at) d[v] = val;
  }
  if (!a.normalize && live) {
    T raw[V];
    float x[V], mx, part = 0.f;
    load_logits<T, V>(reinterpret_cast<const T*>(a.logits) + (long long)t * a.stride, a.G, lane, a.vec != 0, raw);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = Elem<T>::to_f(raw[v]);
    mx = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) mx = fmaxf(mx, x[v]);
    mx = warp_max(mx);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      x[v] = lane * V + v < a.G ? share_of(x[v], mx) : 0.f;
      part += x[v];
    }
    const float inv = 1.f / warp_sum(part);
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] = x[v] * inv * (d[v] - mean);
  }
  T* out = reinterpret_cast<T*>(a.dlogits) + (long long)t * a.G;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane * V + v < a.G) out[lane * V + v] = Elem<T>::from_f(d[v]);
}

void plan(RouteArgs& a) {
  // one block while its warps have few tokens each; then as many blocks as make full waves, in whole mask words
  if (a.N <= 128) {
    a.per_block = 128;
  } else {
    // (seven blocks of eight warps an SM: 32768 tokens of 256 experts 23 us)
    a.per_block = std::min(kMaxPerBlock, std::max(32, (a.N / 1036 + 31) / 32 * 32));
  }
  a.blocks = (a.N + a.per_block - 1) / a.per_block;
}

template <typename T, int V, bool PACKED>
cudaError_t launch_choose(RouteArgs a, cudaStream_t st) {
  // (64 registers to a thread are enough for up to 256 experts)
  constexpr int kAlone = V <= 8 ? 32 : 8;
  const size_t counts = sizeof(int) * a.G, masks = sizeof(unsigned) * a.G * (kMaxPerBlock / 32);
  if (a.blocks <= 1) {
    a.blocks = 1;
    route_choose_kernel<T, V, PACKED, true, kAlone><<<1, 32 * kAlone, counts + masks, st>>>(a);
    count_launch();
    return cudaGetLastError();
  }
  route_choose_kernel<T, V, PACKED, false, kChooseWarps><<<a.blocks, 32 * kChooseWarps, counts, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_early(route_scan_kernel, dim3((a.G + 7) / 8), dim3(256), 0, st, a);
  if (e == cudaSuccess) e = launch_early(route_number_kernel, dim3(a.blocks), dim3(256), counts + masks, st, a);
  count_launch(3);
  return e;
}
template <typename T, int V>
cudaError_t launch_route(const RouteArgs& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (!a.bias) return launch_choose<T, V, true>(a, st);
  }
  return launch_choose<T, V, false>(a, st);
}
template <typename T, int V>
cudaError_t launch_route_bwd(const RouteArgs& a, cudaStream_t st) {
  route_bwd_kernel<T, V><<<(a.N + 7) / 8, 256, 0, st>>>(a);
  count_launch();
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------- combine
// A block takes 256 P packets of a token's column, P to a thread, two of the token's pairs at a time: 2 P loads under way.
template <typename T, int VEC, int P>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a, int chunks) {
  const int t = blockIdx.x / chunks, c0 = (blockIdx.x % chunks) * (256 * P) + threadIdx.x, per = a.E / VEC;
  if (c0 >= per) return;
  const int* position = a.position + (long long)t * a.k;
  const float* weights = a.weights ? a.weights + (long long)t * a.k : nullptr;
  const Pack<T, VEC>* Y = reinterpret_cast<const Pack<T, VEC>*>(a.Y);
  const long long ld = a.Y_stride / VEC;
  float acc[P][VEC];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[p][v] = 0.f;
  for (int j = 0; j < a.k; j += 2) {
    Pack<T, VEC> y[2][P];
    float w[2];
    bool there[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int at = j + u < a.k ? position[j + u] : -1;
      there[u] = at >= 0 && at < a.R;
      w[u] = there[u] && weights ? weights[j + u] : 1.f;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (there[u] && c0 + 256 * p < per) y[u][p] = Y[(long long)at * ld + c0 + 256 * p];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!there[u]) continue;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[p][v] = fmaf(w[u], Elem<T>::to_f(y[u][p].v[v]), acc[p][v]);
    }
  }
  Pack<T, VEC>* out = reinterpret_cast<Pack<T, VEC>*>(reinterpret_cast<T*>(a.y) + (long long)t * a.y_stride);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (c0 + 256 * p >= per) continue;
    Pack<T, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = Elem<T>::from_f(acc[p][v]);
    out[c0 + 256 * p] = o;
  }
}

// A warp takes a column of Y: its token, the weight that names it, the gradient of both.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_bwd_kernel(const CombineArgs a) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= a.R) return;
  const int t = a.columns[r];
  const bool there = t >= 0 && t < a.N;
  float w = 0.f;
  bool named = false;
  if (there) {
    for (int j = 0; j < a.k; ++j) {
      if (a.position[(long long)t * a.k + j] != r) continue;
      named = true;
      w += a.weights ? a.weights[(long long)t * a.k + j] : 1.f;
    }
  }
  T* dY = reinterpret_cast<T*>(a.dY) + (long long)r * a.E;
  if (!named) {
    for (int c = lane; c < a.E; c += 32) dY[c] = Elem<T>::from_f(0.f);
    return;
  }
  const T* dy = reinterpret_cast<const T*>(a.dy) + (long long)t * a.dy_stride;
  const T* Y = reinterpret_cast<const T*>(a.Y) + (long long)r * a.Y_stride;
  float dot = 0.f;
#pragma unroll 4
  for (int c = lane * VEC; c < a.E; c += 32 * VEC) {
    const Pack<T, VEC> d = *reinterpret_cast<const Pack<T, VEC>*>(dy + c);
    Pack<T, VEC> out;
#pragma unroll
    for (int v = 0; v < VEC; ++v) out.v[v] = Elem<T>::from_f(w * Elem<T>::to_f(d.v[v]));
    *reinterpret_cast<Pack<T, VEC>*>(dY + c) = out;
    if (a.dweights) {
      const Pack<T, VEC> y = *reinterpret_cast<const Pack<T, VEC>*>(Y + c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) dot = fmaf(Elem<T>::to_f(d.v[v]), Elem<T>::to_f(y.v[v]), dot);
    }
  }
  if (a.dweights) {
    dot = warp_sum(dot);
    for (int j = lane; j < a.k; j += 32)
      if (a.position[(long long)t * a.k + j] == r) a.dweights[(long long)t * a.k + j] = dot;
  }
}
// zeros for the weights of pairs that combine_bwd_kernel does not meet
__global__ void __launch_bounds__(256) combine_rest_kernel(const CombineArgs a) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.N * a.k) return;
  const int p = a.position[i];
  if (p < 0 || p >= a.R || a.columns[p] != (int)(i / a.k)) a.dweights[i] = 0.f;
}

bool packets(const void* p, long long stride, int bytes, int esize) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (stride * esize) % bytes == 0;
}
template <typename T, int VEC>
cudaError_t launch_combine(const CombineArgs& a, bool bwd, cudaStream_t st) {
  if (!bwd) {
    const int per = a.E / VEC, P = per > 256 ? 2 : 1, chunks = (per + 256 * P - 1) / (256 * P);
    const long long blocks = (long long)chunks * a.N;
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    if (P == 2) combine_kernel<T, VEC, 2><<<(unsigned)blocks, 256, 0, st>>>(a, chunks);
    else combine_kernel<T, VEC, 1><<<(unsigned)blocks, 256, 0, st>>>(a, chunks);
    count_launch();
  } else {
    if (a.R) combine_bwd_kernel<T, VEC><<<(a.R + 7) / 8, 256, 0, st>>>(a);
    const long long pairs = (long long)a.N * a.k;
    if (a.dweights && pairs) combine_rest_kernel<<<(unsigned)((pairs + 255) / 256), 256, 0, st>>>(a);
    count_launch((a.R ? 1 : 0) + (a.dweights && pairs ? 1 : 0));
  }
  return cudaGetLastError();
}
template <typename T>
cudaError_t combine_of(const CombineArgs& a, bool bwd, cudaStream_t st) {
  const int z = sizeof(T);
  const bool whole = packets(a.Y, a.Y_stride, 16, z) && a.E % (16 / z) == 0 &&
                     (bwd ? packets(a.dy, a.dy_stride, 16, z) && packets(a.dY, a.E, 16, z) : packets(a.y, a.y_stride, 16, z));
  return whole ? launch_combine<T, 16 / sizeof(T)>(a, bwd, st) : launch_combine<T, 1>(a, bwd, st);
}

template <typename T>
cudaError_t route_of(RouteArgs a, bool bwd, cudaStream_t st) {
  int v = 1;
  while (32 * v < a.G) v *= 2;
  a.k_up = 1;
  while (a.k_up < a.k) a.k_up *= 2;
  a.vec = packets(a.logits, a.stride, std::min<int>(16, v * sizeof(T)), sizeof(T));
#define NB_V(VV)                                                                          \
  if (a.G <= 32 * VV) return bwd ? launch_route_bwd<T, VV>(a, st) : launch_route<T, VV>(a, st)
  NB_V(1);
  NB_V(2);
  NB_V(4);
  NB_V(8);
  NB_V(16);
  NB_V(32);
#undef NB_V
  return cudaErrorInvalidValue;
}

}  // namespace

size_t route_workspace_bytes(const RouteArgs& a0) {
  RouteArgs a = a0;
  plan(a);
  return a.blocks <= 1 ? 0 : sizeof(int) * (size_t)a.G * (a.blocks + 1);
}
cudaError_t route(RouteArgs a, int dtype, cudaStream_t st) {
  plan(a);
  switch (dtype) {
    case NNLIB_B200_F16:  return route_of<__half>(a, false, st);
    case NNLIB_B200_BF16: return route_of<__nv_bfloat16>(a, false, st);
    default:              return route_of<float>(a, false, st);
  }
}
cudaError_t route_bwd(const RouteArgs& a, int dtype, cudaStream_t st) {
  if (!a.N) return cudaSuccess;
  switch (dtype) {
    case NNLIB_B200_F16:  return route_of<__half>(a, true, st);
    case NNLIB_B200_BF16: return route_of<__nv_bfloat16>(a, true, st);
    default:              return route_of<float>(a, true, st);
  }
}
cudaError_t combine(const CombineArgs& a, int dtype, cudaStream_t st) {
  if (!a.N || !a.E) return cudaSuccess;
  switch (dtype) {
    case NNLIB_B200_F16:  return combine_of<__half>(a, false, st);
    case NNLIB_B200_BF16: return combine_of<__nv_bfloat16>(a, false, st);
    default:              return combine_of<float>(a, false, st);
  }
}
cudaError_t combine_bwd(const CombineArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case NNLIB_B200_F16:  return combine_of<__half>(a, true, st);
    case NNLIB_B200_BF16: return combine_of<__nv_bfloat16>(a, true, st);
    default:              return combine_of<float>(a, true, st);
  }
}

}  // namespace nb200
