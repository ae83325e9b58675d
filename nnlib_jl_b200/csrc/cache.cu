// Tokens into and out of the 8-bit key / value cache (nnlib_b200.h: pages, scales, codes).
//
// Write: one block for a page that a sequence's new tokens touch, a head, and keys or values.  It is the only one that
// touches this page's scale and codes of this head, so there is nothing to order: it finds the new tokens' largest
// magnitude, settles the scale, rounds the older codes anew where the scale has grown, and writes the new ones.
// Read: 16 codes to a thread.  Both are bound by HBM: an element is two bytes on one side and one on the other.
#include <algorithm>

#include "cache_codes.cuh"

namespace nb200 {
namespace {

constexpr int kWrThreads = 256;

template <typename T, int CODE>
__global__ void __launch_bounds__(kWrThreads) cache_write_kernel(const CacheArgs c, const CacheTokens t) {
  __shared__ float sm[kWrThreads / 32];
  const int kv = blockIdx.y / c.H, h = blockIdx.y % c.H, b = blockIdx.z, tid = threadIdx.x;
  const int T_ = 1 << c.log_page;
  const long long start = t.start ? (long long)t.start[b] : t.start0;
  const long long n_new = t.count ? min(max(t.count[b], 0), t.L) : t.L;
  if (start < 0) return;
  const long long p = (start >> c.log_page) + blockIdx.x;              // page of the sequence
  if (p >= c.rows) return;
  const long long lo = max(start, p << c.log_page), hi = min(start + n_new, (p + 1) << c.log_page);
  if (lo >= hi) return;
  const long long page = cache_page(c, b, p);
  if (page < 0) return;
  const int fill = (int)(lo - (p << c.log_page)), n = (int)(hi - lo);  // older tokens of the page, new ones
  const T* x = reinterpret_cast<const T*>(t.x[kv]) + (lo - start) * t.sl[kv] + b * t.sb[kv] + (long long)h * c.d;
  unsigned char* codes = c.codes[kv] + (page * T_) * c.row + (long long)h * c.d;
  float* scale = c.scale[kv] + page * c.H + h;

  float amax = 0.f;
  bool bad = false;
  for (int i = tid; i < n * c.d; i += kWrThreads) {
    const int l = i / c.d, e = i - l * c.d;
    const float v = fabsf(Elem<T>::to_f(x[l * t.sl[kv] + e]));
    bad |= !(v <= 3.402823466e38f);
    amax = fmaxf(amax, v);
  }
  if (bad) amax = __int_as_float(0x7f800000);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if ((tid & 31) == 0) sm[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWrThreads / 32; ++w) amax = fmaxf(amax, sm[w]);

  const float old = fill > 0 ? *scale : 0.f;
  const float asked = block_scale<CODE>(amax);
  const float s = (old != old || asked != asked) ? __int_as_float(0x7fc00000) : fmaxf(old, asked);
  const float inv = inverse_scale(s);
  if (fill > 0 && s > old) {
    const float f = __fdiv_rn(old, s);
    for (int i = tid; i < fill * c.d; i += kWrThreads) {
      const int l = i / c.d, e = i - l * c.d;
      unsigned char* q = codes + l * c.row + e;
      *q = (unsigned char)to_code<CODE>(from_code<CODE>(*q), f);
    }
  }
  for (int i = tid; i < n * c.d; i += kWrThreads) {
    const int l = i / c.d, e = i - l * c.d;
    codes[(fill + l) * c.row + e] = (unsigned char)to_code<CODE>(code_input(Elem<T>::to_f(x[l * t.sl[kv] + e]), inv), inv);
  }
  __syncthreads();                                                     // every thread has read the old scale
  if (tid == 0) *scale = s;
}

template <typename T, int CODE>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheArgs c, const CacheTokens t) {
  const int kv = blockIdx.y, b = blockIdx.z;
  const long long parts = c.row / 16, i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long l = i / parts;
  if (l >= t.L) return;
  const int e0 = (int)(i - l * parts) * 16, h = e0 / c.d;
  const long long pos = l + (t.start ? (long long)t.start[b] : t.start0);
  T out[16];
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  float s = 0.f;
  if (pos >= 0 && pos < (c.rows << c.log_page) && !(t.lens && pos >= t.lens[b])) {
    const long long page = cache_page(c, b, pos >> c.log_page);
    s = __int_as_float(0x7fc00000);
    if (page >= 0) {
      const long long slot = (page << c.log_page) + (pos & ((1 << c.log_page) - 1));
      raw = __ldcs(reinterpret_cast<const uint4*>(c.codes[kv] + slot * c.row + e0));
      s = c.scale[kv][page * c.H + h];
    }
  }
  const unsigned int w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 16; ++j) out[j] = Elem<T>::from_f(from_code<CODE>(w[j >> 2] >> (8 * (j & 3))) * s);
  T* y = reinterpret_cast<T*>(t.x[kv]) + l * t.sl[kv] + b * t.sb[kv] + e0;
  if (((reinterpret_cast<uintptr_t>(y) & 15u) == 0)) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(out) / 16; ++j) {
      uint4 v;
      memcpy(&v, reinterpret_cast<const char*>(out) + 16 * j, 16);
      reinterpret_cast<uint4*>(y)[j] = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = out[j];
  }
}

template <typename T>
cudaError_t write_t(const CacheArgs& c, const CacheTokens& t, cudaStream_t st) {
  const int T_ = 1 << c.log_page;
  const long long pages = std::min<long long>((t.L + T_ - 2) / T_ + 1, c.rows);    // that L tokens can touch
  const dim3 grid((unsigned)pages, 2 * c.H, c.B);
  if (c.code == NNLIB_B200_INT8) cache_write_kernel<T, NNLIB_B200_INT8><<<grid, kWrThreads, 0, st>>>(c, t);
  else cache_write_kernel<T, NNLIB_B200_E4M3><<<grid, kWrThreads, 0, st>>>(c, t);
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t read_t(const CacheArgs& c, const CacheTokens& t, cudaStream_t st) {
  const long long items = (long long)t.L * (c.row / 16);
  const dim3 grid((unsigned)((items + 255) / 256), 2, c.B);
  if (c.code == NNLIB_B200_INT8) cache_read_kernel<T, NNLIB_B200_INT8><<<grid, 256, 0, st>>>(c, t);
  else cache_read_kernel<T, NNLIB_B200_E4M3><<<grid, 256, 0, st>>>(c, t);
  count_launch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t cache_write(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st) {
  if (dtype == NNLIB_B200_F16) return write_t<__half>(c, t, st);
  if (dtype == NNLIB_B200_BF16) return write_t<__nv_bfloat16>(c, t, st);
  return write_t<float>(c, t, st);
}

cudaError_t cache_read(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st) {
  if (dtype == NNLIB_B200_F16) return read_t<__half>(c, t, st);
  if (dtype == NNLIB_B200_BF16) return read_t<__nv_bfloat16>(c, t, st);
  return read_t<float>(c, t, st);
}

}  // namespace nb200
