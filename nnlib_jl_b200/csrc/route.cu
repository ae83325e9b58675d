// The router of a layer of experts and the sum that ends it (include/nnlib_b200.h: nnlib_b200_route, nnlib_b200_combine).
//
// route: S_t = the k largest of l_t + b; w = softmax(l) over S_t or over all; then a stable counting sort of the chosen
// (token, expert) pairs by expert.  A warp takes a token, its G logits as order-preserving integers in registers, and picks
// the largest k times (redux.sync gives a warp's largest; the first lane that has it has the lowest expert, since lanes hold
// neighbouring experts).  A block counts its tokens' choices; a second launch turns the counts of all blocks into each
// block's first number for each expert; a third gives every pair its number: a token picks an expert at most once, so the
// pair's place among its block's is the number of earlier tokens in the expert's bit mask.  Nothing depends on the order in
// which warps run.  Few tokens take one block and one launch.
//
// combine: HBM bound, 16 bytes a thread and column.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kChooseWarps = 16;
constexpr int kMaxPerBlock = 256;        // tokens whose choices one block numbers: the masks of an expert are 8 words

// Larger floats are larger integers; -0 like +0; NaN below everything, 0 for what cannot be chosen.
__device__ __forceinline__ unsigned sortable(float x) {
  if (isnan(x)) return 1u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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

// V neighbouring logits of a token for each lane; -Inf where there is no expert
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* row, int G, int lane, float (&x)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    x[v] = e < G ? Elem<T>::to_f(row[e]) : __int_as_float(0xff800000);
  }
}
// the exponential of a logit relative to the largest: the slow branch of the softmax for +Inf
__device__ __forceinline__ float share_of(float x, float mx) {
  if (mx == __int_as_float(0x7f800000)) return x == mx ? 1.f : (isnan(x) ? x : 0.f);
  return expf(x - mx);
}

template <typename T, int V>
__device__ void choose_token(const RouteArgs& a, int t, int lane, int* count) {
  const bool live = !a.mask || a.mask[t];
  int mine = -1;                          // lane j: the j-th expert of the token
  float w = 0.f;
  if (live) {
    float x[V];
    load_logits<T, V>(reinterpret_cast<const T*>(a.logits) + (long long)t * a.stride, a.G, lane, x);
    unsigned key[V], best = 0u;
    int at = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      key[v] = e < a.G ? sortable(a.bias ? x[v] + a.bias[e] : x[v]) : 0u;
      if (key[v] > best) { best = key[v]; at = v; }
    }
    float logit = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const unsigned top = __reduce_max_sync(kFull, best);
      const int src = __ffs(__ballot_sync(kFull, best == top)) - 1;
      float mylogit = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v == at) mylogit = x[v];
      const int e = __shfl_sync(kFull, lane * V + at, src);
      const float l = __shfl_sync(kFull, mylogit, src);
      if (lane == j) { mine = e; logit = l; }
      if (lane == src) {
        best = 0u;
        const int gone = at;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (v == gone) key[v] = 0u;
          if (key[v] > best) { best = key[v]; at = v; }
        }
      }
    }
    float mx, part = 0.f;
    if (a.normalize) {
      mx = warp_max(lane < a.k ? logit : __int_as_float(0xff800000));
      if (lane < a.k) part = share_of(logit, mx);
      w = part / warp_sum(part);
    } else {
      mx = x[0];
#pragma unroll
      for (int v = 1; v < V; ++v) mx = fmaxf(mx, x[v]);
      mx = warp_max(mx);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane * V + v < a.G) part += share_of(x[v], mx);
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
template <typename T, int V, bool ALONE>
__global__ void __launch_bounds__(32 * kChooseWarps) route_choose_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  __shared__ int part[kChooseWarps];
  const int t0 = blockIdx.x * a.per_block, t1 = min(a.N, t0 + a.per_block);
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  for (int t = t0 + (threadIdx.x >> 5); t < t1; t += kChooseWarps) choose_token<T, V>(a, t, threadIdx.x & 31, sm);
  __syncthreads();
  if constexpr (ALONE) {
    const int total = block_scan<kChooseWarps>(sm, a.G, part);
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
  if (e >= a.G) return;
  int* c = a.ws + (long long)e * a.blocks;
  int carry = 0;
  for (int i0 = 0; i0 < a.blocks; i0 += 32) {
    const int own = i0 + lane < a.blocks ? c[i0 + lane] : 0;
    int s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += u;
    }
    if (i0 + lane < a.blocks) c[i0 + lane] = carry + s - own;
    carry += __shfl_sync(kFull, s, 31);
  }
  if (lane == 0) a.ws[(long long)a.G * a.blocks + e] = carry;
}

__global__ void __launch_bounds__(512) route_number_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  __shared__ int part[16];
  const int* totals = a.ws + (long long)a.G * a.blocks;
  for (int i = threadIdx.x; i < a.G; i += blockDim.x) sm[i] = totals[i];
  __syncthreads();
  const int total = block_scan<16>(sm, a.G, part);
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
    float x[V], mx, part = 0.f;
    load_logits<T, V>(reinterpret_cast<const T*>(a.logits) + (long long)t * a.stride, a.G, lane, x);
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
  // one block while its warps have few tokens each; then as many blocks as keep every SM busy, in whole mask words
  if (a.N <= 128) {
    a.per_block = 128;
  } else {
    a.per_block = std::min(kMaxPerBlock, std::max(32, (a.N / 296 + 31) / 32 * 32));
  }
  a.blocks = (a.N + a.per_block - 1) / a.per_block;
}

template <typename T, int V>
cudaError_t launch_route(RouteArgs a, cudaStream_t st) {
  const size_t counts = sizeof(int) * a.G, masks = sizeof(unsigned) * a.G * (kMaxPerBlock / 32);
  if (a.blocks <= 1) {
    a.blocks = 1;
    route_choose_kernel<T, V, true><<<1, 32 * kChooseWarps, counts + masks, st>>>(a);
    count_launch();
    return cudaGetLastError();
  }
  route_choose_kernel<T, V, false><<<a.blocks, 32 * kChooseWarps, counts, st>>>(a);
  route_scan_kernel<<<(a.G + 7) / 8, 256, 0, st>>>(a);
  route_number_kernel<<<a.blocks, 512, counts + masks, st>>>(a);
  count_launch(3);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t launch_route_bwd(const RouteArgs& a, cudaStream_t st) {
  route_bwd_kernel<T, V><<<(a.N + 7) / 8, 256, 0, st>>>(a);
  count_launch();
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------- combine
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  const int per = a.E / VEC;               // packets of a column
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)per * a.N) return;
  const int t = (int)(i / per), c = (int)(i % per) * VEC;
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const int p = a.position[(long long)t * a.k + j];
    if (p < 0 || p >= a.R) continue;
    const float w = a.weights ? a.weights[(long long)t * a.k + j] : 1.f;
    const Pack<T, VEC> y = *reinterpret_cast<const Pack<T, VEC>*>(reinterpret_cast<const T*>(a.Y) + (long long)p * a.Y_stride + c);
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w, Elem<T>::to_f(y.v[v]), acc[v]);
  }
  Pack<T, VEC> out;
#pragma unroll
  for (int v = 0; v < VEC; ++v) out.v[v] = Elem<T>::from_f(acc[v]);
  *reinterpret_cast<Pack<T, VEC>*>(reinterpret_cast<T*>(a.y) + (long long)t * a.y_stride + c) = out;
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
    const long long n = (long long)(a.E / VEC) * a.N, blocks = (n + 255) / 256;
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    combine_kernel<T, VEC><<<(unsigned)blocks, 256, 0, st>>>(a);
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
cudaError_t route_of(const RouteArgs& a, bool bwd, cudaStream_t st) {
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
