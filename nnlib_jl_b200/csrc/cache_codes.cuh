// The 8-bit cache's pages, scales and codes (nnlib_b200.h), as its kernels see them.
#pragma once

#include "common.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr float kScaleTiny = 1.17549435e-38f;     // 2^-126: a smaller scale is none

// Page number p of sequence b; -1: none, or one that the pool does not have.
__device__ __forceinline__ long long cache_page(const CacheArgs& c, int b, long long p) {
  const long long n = c.table ? (long long)c.table[p + c.table_stride * b] : c.run * b + p;
  return (n >= 0 && n < c.pages) ? n : -1;
}

// The scale that a block asks for whose largest magnitude is amax; NaN for one that is not finite.
template <int CODE>
__device__ __forceinline__ float block_scale(float amax) {
  if (!(amax <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
  float s;
  if (CODE == NNLIB_B200_INT8) {
    s = __fmul_rn(amax, 1.f / 127.f);    // (the constant rounded to Float32)
  } else {
    // 2^e with 448 * 2^e >= amax, 448 = 0.875 * 2^9
    int e;
    const float m = frexpf(amax, &e);
    s = ldexpf(1.f, e - 9 + (m > 0.875f ? 1 : 0));
  }
  return (amax > 0.f && s >= kScaleTiny) ? s : 0.f;
}

// Four x / scale as codes, given 1 / scale.  No x is larger than 127 or 448 scales but for the rounding of the inverse, less
// than half a code.  Int8: rounded by adding 1.5 * 2^23, whose last byte is then the code (the conversion instruction runs
// at a quarter of the rate).
template <int CODE>
__device__ __forceinline__ uint32_t to_codes4(float a, float b, float c, float d, float inv) {
  if (CODE == NNLIB_B200_INT8) {
    auto bits = [&](float x) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); };
    return __byte_perm(__byte_perm(bits(a), bits(b), 0x0040u), __byte_perm(bits(c), bits(d), 0x0040u), 0x5410u);
  }
  auto pair = [&](float x, float y) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(__fmul_rn(y, inv)), "f"(__fmul_rn(x, inv)));
    return (uint32_t)r;
  };
  return pair(a, b) | (pair(c, d) << 16);
}

// the four numbers that the codes of a word are
template <int CODE>
__device__ __forceinline__ void from_codes4(uint32_t w, float (&f)[4]) {
  if (CODE == NNLIB_B200_INT8) {
    // code + 128 as the last byte of 2^23
    const uint32_t u = w ^ 0x80808080u;
    f[0] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440u)) - 8388736.f;
    f[1] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441u)) - 8388736.f;
    f[2] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442u)) - 8388736.f;
    f[3] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443u)) - 8388736.f;
  } else {
    uint32_t lo, hi;
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
    __half2 h;
    memcpy(&h, &lo, 4);
    f[0] = __low2float(h);
    f[1] = __high2float(h);
    memcpy(&h, &hi, 4);
    f[2] = __low2float(h);
    f[3] = __high2float(h);
  }
}

__device__ __forceinline__ float inverse_scale(float s) { return s > 0.f ? __fdiv_rn(1.f, s) : 0.f; }

}  // namespace
}  // namespace nb200
