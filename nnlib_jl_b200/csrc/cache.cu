// Tokens into and out of the 8-bit key / value cache (nnlib_b200.h: pages, scales, codes).
//
// Both are bound by HBM: an element is two bytes (or four) on one side and one on the other.  (32768 bf16 tokens of 8 heads of
// 128 into pages of 64: written in 36 us, 5.5 TB/s, read back in 40 us, 5.0 TB/s.  More in flight to a thread, half the
// blocks: 46 and 49.)
// Write: one block for a page that a sequence's new tokens touch, a head, and keys or values.  It is the only one that
// touches this page's scale and codes of this head, so there is nothing to order: it finds the new tokens' largest
// magnitude, settles the scale, rounds the older codes anew where the scale has grown, and writes the new ones.  A thread
// works on 16 bytes of elements at a time and keeps the first kHeld such pieces in registers between the two steps; blocks
// of more (pages of more than 16384 16-bit elements of a head) read the rest again, from L2.
// Read: eight codes to a thread and store, so that a warp's stores of 16-bit results are whole lines.
#include <algorithm>

#include "cache_codes.cuh"

namespace nb200 {
namespace {

constexpr int kHeld = 8;                  // pieces of 16 bytes that a thread keeps

// 16 bytes of elements; VEC: in one load
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_piece(const T* p) {
  if constexpr (VEC) return __ldcs(reinterpret_cast<const uint4*>(p));
  uint32_t w[4];
  if constexpr (sizeof(T) == 2) {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = q[2 * i] | ((uint32_t)q[2 * i + 1] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest magnitude so far, as bits: of Float32, or two by two of 16-bit numbers.  As whole numbers magnitudes keep their
// order, and a NaN is larger than all others.
template <typename T>
__device__ __forceinline__ uint32_t magnitude(uint32_t top, const uint4& v) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t m = 0x7fff7fffu;
    return __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m)));
  } else {
    const uint32_t m = 0x7fffffffu;
    return max(top, max(max(v.x & m, v.y & m), max(v.z & m, v.w & m)));
  }
}

__device__ __forceinline__ float2 two_floats(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 two_floats(uint32_t w, __half) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}

// (an argument indexed by a number that is not a constant would be copied to local memory whole)
template <typename X>
__device__ __forceinline__ X pick(const X (&v)[2], int kv) { return kv ? v[1] : v[0]; }

template <typename T, int CODE, bool VEC>
__global__ void __launch_bounds__(256, 3) cache_write_kernel(const CacheArgs c, const CacheTokens t) {
  constexpr int U = 16 / sizeof(T);        // elements of a piece: as many bytes of codes
  __shared__ uint32_t sm[8];
  // heads side by side: what runs at one time reads whole tokens
  const int h = blockIdx.x % c.H, kv = (blockIdx.x / c.H) & 1, b = blockIdx.y, tid = threadIdx.x, nt = blockDim.x;
  const long long start = t.start ? (long long)t.start[b] : t.start0;
  const long long n_new = t.count ? min(max(t.count[b], 0), t.L) : t.L;
  if (start < 0) return;
  const long long p = (start >> c.log_page) + blockIdx.x / (2 * c.H);  // page of the sequence
  if (p >= c.rows) return;
  const long long lo = max(start, p << c.log_page), hi = min(start + n_new, (p + 1) << c.log_page);
  if (lo >= hi) return;
  const int fill = (int)(lo - (p << c.log_page));                      // older tokens of the page
  const unsigned pieces = c.d / U, n = (unsigned)(hi - lo) * pieces;   // new ones, in pieces
  const long long sl = pick(t.sl, kv);
  const T* x = reinterpret_cast<const T*>(pick(t.x, kv)) + (lo - start) * sl + b * pick(t.sb, kv) + (long long)h * c.d;
  // where pieces tid, tid + nt, ... are: token, piece of the token
  const unsigned l0 = tid / pieces, e0 = tid - l0 * pieces, dl = nt / pieces, de = nt - dl * pieces;
  auto advance = [&](unsigned& l, unsigned& e) {
    l += dl;
    e += de;
    if (e >= pieces) e -= pieces, ++l;
  };
  auto source = [&](unsigned l, unsigned e) { return x + (long long)l * sl + e * U; };

  uint4 held[kHeld];
  unsigned l = l0, e = e0;
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    held[r] = make_uint4(0u, 0u, 0u, 0u);
    if (tid + r * nt < n) held[r] = load_piece<T, VEC>(source(l, e));
    advance(l, e);
  }
  const long long page = cache_page(c, b, p);
  if (page < 0) return;
  unsigned char* codes = pick(c.codes, kv) + (page << c.log_page) * c.row + (long long)h * c.d;
  float* scale = pick(c.scale, kv) + page * c.H + h;
  const float old = fill > 0 ? *scale : 0.f;

  uint32_t top = 0u;
#pragma unroll
  for (int r = 0; r < kHeld; ++r) top = magnitude<T>(top, held[r]);
  for (unsigned i = tid + kHeld * nt; i < n; i += nt, advance(l, e)) top = magnitude<T>(top, load_piece<T, VEC>(source(l, e)));
  if constexpr (sizeof(T) == 2) {
    top = max(top >> 16, top & 0xffffu);
    top = __float_as_uint(two_floats(top, T()).x);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (nt > 32) {
    if ((tid & 31) == 0) sm[tid >> 5] = top;
    __syncthreads();
    for (int w = 0; w < nt / 32; ++w) top = max(top, sm[w]);
  }

  const float asked = block_scale<CODE>(__uint_as_float(top));
  const float s = (old != old || asked != asked) ? __int_as_float(0x7fc00000) : fmaxf(old, asked);
  const float inv = inverse_scale(s);
  if (fill > 0 && s > old) {
    const float f = __fdiv_rn(old, s);               // (0 where the older codes are all 0)
    const unsigned per = c.d / 16;
    for (unsigned i = tid; i < fill * per; i += nt) {
      uint4* q = reinterpret_cast<uint4*>(codes + (long long)(i / per) * c.row + (i % per) * 16);
      uint4 v = *q;
      auto again = [&](uint32_t w) {
        float g[4];
        from_codes4<CODE>(w, g);
        return to_codes4<CODE>(g[0], g[1], g[2], g[3], f);
      };
      *q = make_uint4(again(v.x), again(v.y), again(v.z), again(v.w));
    }
  }
  unsigned char* to0 = codes + (long long)fill * c.row;
  auto quantise = [&](const uint4& v) {
    unsigned char* to = to0 + (long long)l * c.row + e * U;
    if constexpr (sizeof(T) == 2) {
      const float2 a = two_floats(v.x, T()), b2 = two_floats(v.y, T()), c2 = two_floats(v.z, T()), d2 = two_floats(v.w, T());
      *reinterpret_cast<uint2*>(to) = make_uint2(to_codes4<CODE>(a.x, a.y, b2.x, b2.y, inv), to_codes4<CODE>(c2.x, c2.y, d2.x, d2.y, inv));
    } else {
      *reinterpret_cast<uint32_t*>(to) = to_codes4<CODE>(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w), inv);
    }
  };
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  if (inv == 0.f) {                      // a scale of 0 or NaN: all codes are 0, also of what is not finite
#pragma unroll
    for (int r = 0; r < kHeld; ++r) held[r] = zero;
  }
  l = l0;
  e = e0;
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    if (tid + r * nt < n) quantise(held[r]);
    advance(l, e);
  }
  for (unsigned i = tid + kHeld * nt; i < n; i += nt, advance(l, e))
    quantise(inv == 0.f ? zero : load_piece<T, VEC>(source(l, e)));
  // (every thread has read the old scale: it came before the barrier, or the block is one warp)
  if (tid == 0) *scale = s;
}

constexpr int kReadTokens = 16;            // tokens of a block: never more than a page's

// VEC: results may be stored 16 bytes at a time
template <typename T, int CODE, bool VEC>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheArgs c, const CacheTokens t) {
  const int kv = blockIdx.y & 1, b = blockIdx.y >> 1;
  const int parts = (int)(c.row / 8), width = min(parts, 256), rows = 256 / width;   // eight codes to a thread, tokens side by side
  const int col = threadIdx.x % width, first = threadIdx.x / width;
  const long long start = t.start ? (long long)t.start[b] : t.start0;
  // the block's tokens are those of one aligned sixteen, so one page's (below zero, too)
  const long long p16 = (start >> 4) + blockIdx.x, lo = max(p16 << 4, start), hi = min((p16 + 1) << 4, start + t.L);
  const long long cap = c.rows << c.log_page, end = t.lens ? min(cap, (long long)t.lens[b]) : cap;
  const bool inside = lo >= 0 && lo < end;
  const long long page = inside ? cache_page(c, b, lo >> c.log_page) : -1;
  const unsigned char* codes = pick(c.codes, kv) + (page < 0 ? 0 : ((page << c.log_page) + (lo & ((1 << c.log_page) - 1))) * c.row);
  T* y = reinterpret_cast<T*>(pick(t.x, kv)) + (lo - start) * pick(t.sl, kv) + b * pick(t.sb, kv);
  const float* scale = pick(c.scale, kv);
  const long long sl_y = pick(t.sl, kv);
  const int n = (int)(hi - lo), n_in = inside ? (int)min((long long)n, end - lo) : 0;
  if (first >= rows) return;
  for (int part = col; part < parts; part += width) {
    float s = __int_as_float(0x7fc00000);
    if (page >= 0) s = scale[page * c.H + part * 8 / c.d];
#pragma unroll 4
    for (int l = first; l < n; l += rows) {
      uint2 raw = make_uint2(0u, 0u);
      if (l < n_in && page >= 0) raw = __ldcs(reinterpret_cast<const uint2*>(codes + l * c.row + part * 8));
      const float sl = l < n_in ? s : 0.f;
      float f[8];
      {
        float lo4[4], hi4[4];
        from_codes4<CODE>(raw.x, lo4);
        from_codes4<CODE>(raw.y, hi4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = lo4[e] * sl;
          f[4 + e] = hi4[e] * sl;
        }
      }
      T out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = Elem<T>::from_f(f[e]);
      T* to = y + l * sl_y + part * 8;
      if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < (int)sizeof(out) / 16; ++e) {
          uint4 v;
          memcpy(&v, reinterpret_cast<const char*>(out) + 16 * e, 16);
          __stcs(reinterpret_cast<uint4*>(to) + e, v);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = out[e];
      }
    }
  }
}

// may elements be moved 16 bytes at a time?
bool vectors(const CacheTokens& t, int esize) {
  for (int i = 0; i < 2; ++i)
    if (reinterpret_cast<uintptr_t>(t.x[i]) % 16 || t.sl[i] * esize % 16 || t.sb[i] * esize % 16) return false;
  return true;
}

template <typename T, int CODE>
cudaError_t write_t(const CacheArgs& c, const CacheTokens& t, cudaStream_t st) {
  const int T_ = 1 << c.log_page;
  const long long pages = std::min<long long>((t.L + T_ - 2) / T_ + 1, c.rows);    // that L tokens can touch
  if (pages * 2 * c.H > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)(pages * 2 * c.H), c.B);
  const int pieces = std::min(t.L, T_) * c.d / (16 / (int)sizeof(T));
  const int threads = std::min(256, std::max(32, (pieces / kHeld + 31) & ~31));
  if (vectors(t, sizeof(T))) cache_write_kernel<T, CODE, true><<<grid, threads, 0, st>>>(c, t);
  else cache_write_kernel<T, CODE, false><<<grid, threads, 0, st>>>(c, t);
  count_launch();
  return cudaGetLastError();
}

template <typename T, int CODE>
cudaError_t read_t(const CacheArgs& c, const CacheTokens& t, cudaStream_t st) {
  const dim3 grid((unsigned)((t.L + kReadTokens - 2) / kReadTokens + 1), 2 * c.B);   // aligned sixteens that L tokens touch
  if (vectors(t, sizeof(T))) cache_read_kernel<T, CODE, true><<<grid, 256, 0, st>>>(c, t);
  else cache_read_kernel<T, CODE, false><<<grid, 256, 0, st>>>(c, t);
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t move_t(const CacheArgs& c, const CacheTokens& t, bool in, cudaStream_t st) {
  if (c.code == NNLIB_B200_INT8) return in ? write_t<T, NNLIB_B200_INT8>(c, t, st) : read_t<T, NNLIB_B200_INT8>(c, t, st);
  return in ? write_t<T, NNLIB_B200_E4M3>(c, t, st) : read_t<T, NNLIB_B200_E4M3>(c, t, st);
}

cudaError_t move(const CacheArgs& c, const CacheTokens& t, int dtype, bool in, cudaStream_t st) {
  if (dtype == NNLIB_B200_F16) return move_t<__half>(c, t, in, st);
  if (dtype == NNLIB_B200_BF16) return move_t<__nv_bfloat16>(c, t, in, st);
  return move_t<float>(c, t, in, st);
}

}  // namespace

cudaError_t cache_write(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st) { return move(c, t, dtype, true, st); }
cudaError_t cache_read(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st) { return move(c, t, dtype, false, st); }

}  // namespace nb200
