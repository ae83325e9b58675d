// The 8-bit cache's pages, scales and codes (nnlib_b200.h), as its kernels see them.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr float kScaleTiny = 1.17549435e-38f;     // 2^-126: a smaller scale is none

// Page number p of sequence b; -1: none, or one that the pool does not have.
__device__ __forceinline__ long long cache_page(const CacheArgs& c, int b, long long p) {
  const long long n = c.table ? (long long)c.table[p + c.table_stride * b] : c.rows * b + p;
  return (n >= 0 && n < c.pages) ? n : -1;
}

// The scale that a block asks for whose largest magnitude is amax; NaN for one that is not finite.
template <int CODE>
__device__ __forceinline__ float block_scale(float amax) {
  if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
  float s;
  if (CODE == NNLIB_B200_INT8) {
    s = __fdiv_rn(amax, 127.f);
  } else {
    // 2^e with 448 * 2^e >= amax, 448 = 0.875 * 2^9
    int e;
    const float m = frexpf(amax, &e);
    s = ldexpf(1.f, e - 9 + (m > 0.875f ? 1 : 0));
  }
  return (amax > 0.f && s >= kScaleTiny) ? s : 0.f;
}

// x / scale, given 1 / scale (0 for the scales 0 and NaN), as a code's bits
template <int CODE>
__device__ __forceinline__ unsigned int to_code(float x, float inv) {
  const float t = x * inv;
  if (CODE == NNLIB_B200_INT8) return (unsigned int)__float2int_rn(fminf(fmaxf(t, -127.f), 127.f)) & 0xffu;
  return __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
}
// (a product with 0 that is NaN, from an infinity in a block whose scale is NaN, becomes code 0)
__device__ __forceinline__ float code_input(float x, float inv) { return inv == 0.f ? 0.f : x; }

template <int CODE>
__device__ __forceinline__ float from_code(unsigned int bits) {
  if (CODE == NNLIB_B200_INT8) return (float)(signed char)(bits & 0xffu);
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(bits & 0xffu), __NV_E4M3)));
}

__device__ __forceinline__ float inverse_scale(float s) { return s > 0.f ? __fdiv_rn(1.f, s) : 0.f; }

}  // namespace
}  // namespace nb200
