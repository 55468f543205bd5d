// fa4d_cache8.cuh — codes and scales of caches held in 8 bits.
//
// A value is its code times its block's scale.  Scales are powers of two: a code's value then has no
// more bits than the code and is exact in bf16; e4m3 codes have 4 bits whatever the scale, and keep
// them when their block's scale grows (down to e4m3's subnormals, 2^-15 of the largest); int8 loses
// at most one of its 8 bits against the scale that fits best.
#pragma once

#include <cuda_fp16.h>

#include "fa4d.h"
#include "fa4d_ptx.cuh"

namespace fa4d {

// The four codes of a word to fp16 (exact: e4m3 has 4 significant bits and exponents -9 to 8, int8 7
// and a sign): a = codes 0 and 1, b = codes 2 and 3.
template <bool kInt8>
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (kInt8) {
    // 0x6400 is 1024 in fp16, whose last place is 1: the bytes code + 128 under it make 1152 + code.
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), off), q = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    a = *reinterpret_cast<const uint32_t*>(&p);
    b = *reinterpret_cast<const uint32_t*>(&q);
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
}
template <bool kInt8>
__device__ __forceinline__ void codes_to_float(uint32_t w, float (&f)[4]) {
  uint32_t a, b;
  codes_to_half2<kInt8>(w, a, b);
  const float2 u = unpack2<false>(a), v = unpack2<false>(b);
  f[0] = u.x, f[1] = u.y, f[2] = v.x, f[3] = v.y;
}

// The code nearest to x, ties to even; |x| is at most the largest code.
template <bool kInt8>
__device__ __forceinline__ uint32_t to_code(float x) {
  if constexpr (kInt8) {
    return static_cast<uint32_t>(__float2int_rn(x)) & 0xffu;
  } else {
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(0.f), "f"(x));
    return c & 0xffu;
  }
}
template <bool kInt8>
__device__ __forceinline__ uint32_t to_codes(float x0, float x1, float x2, float x3) {
  if constexpr (kInt8) {
    return to_code<true>(x0) | to_code<true>(x1) << 8 | to_code<true>(x2) << 16 | to_code<true>(x3) << 24;
  } else {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x1), "f"(x0));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x3), "f"(x2));
    return lo | static_cast<uint32_t>(hi) << 16;
  }
}

// The least scale 2^e, e >= -126, under which the magnitude with these bits does not pass the
// largest code: 448 = 1.75 * 2^8 or 127 = 1.984375 * 2^6.  A significand above that one's carries
// into the exponent.  NaN for a magnitude that is not finite.
template <bool kInt8>
__device__ __forceinline__ float least_scale(uint32_t bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  const int e = static_cast<int>((bits + (kInt8 ? 0x01ffffu : 0x1fffffu)) >> 23) - (kInt8 ? 6 : 8);  // biased
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

}  // namespace fa4d
