// fa4d_rotary.cuh — a head's elements as the rotary kernels divide them over threads, and their
// turn.
#pragma once

#include "fa4d.h"
#include "fa4d_ptx.cuh"

namespace fa4d {

// VEC pairs of one head: two runs of VEC elements.  VEC = 8 moves them as two 16-byte
// vectors; VEC = 1 serves sizes and addresses that are not multiples of 16 bytes.
template <int VEC>
struct Run;
template <>
struct Run<8> {
  using T = uint4;
  static __device__ __forceinline__ T load(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void store(uint16_t* p, const T& v) { *reinterpret_cast<uint4*>(p) = v; }
};
template <>
struct Run<1> {
  using T = uint16_t;
  static __device__ __forceinline__ T load(const uint16_t* p) { return *p; }
  static __device__ __forceinline__ void store(uint16_t* p, const T& v) { *p = v; }
};

template <bool kBF16>
__device__ __forceinline__ float to_f(uint16_t x) {
  return unpack2<kBF16>(x).x;
}
template <bool kBF16>
__device__ __forceinline__ uint16_t to_h(float x) {
  return static_cast<uint16_t>(pack2<kBF16>(x, 0.f));
}

// The pair (a, b) turned by the angle of cosine c and sine s.  The products are fused as written, so
// that both widths round alike (left to the compiler, one in 50000 bf16 results differed).
__device__ __forceinline__ float2 turned(float a, float b, float c, float s) {
  return make_float2(fmaf(a, c, -(b * s)), fmaf(b, c, a * s));
}

// Turns the pairs of two runs.  kAdj: the runs are consecutive and pair j is elements
// 2j, 2j+1 of both; otherwise pair j is element j of each.
template <bool kBF16, bool kAdj>
__device__ __forceinline__ void turn(uint4& x, uint4& y, const float (&c)[8], const float (&s)[8]) {
  uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
  uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 a = unpack2<kBF16>(xw[w]), b = unpack2<kBF16>(yw[w]);
    if (kAdj) {
      const float2 u = turned(a.x, a.y, c[w], s[w]), v = turned(b.x, b.y, c[w + 4], s[w + 4]);
      xw[w] = pack2<kBF16>(u.x, u.y);
      yw[w] = pack2<kBF16>(v.x, v.y);
    } else {
      const float2 u = turned(a.x, b.x, c[2 * w], s[2 * w]), v = turned(a.y, b.y, c[2 * w + 1], s[2 * w + 1]);
      xw[w] = pack2<kBF16>(u.x, v.x);
      yw[w] = pack2<kBF16>(u.y, v.y);
    }
  }
}
template <bool kBF16, bool kAdj>
__device__ __forceinline__ void turn(uint16_t& x, uint16_t& y, const float (&c)[1], const float (&s)[1]) {
  const float2 u = turned(to_f<kBF16>(x), to_f<kBF16>(y), c[0], s[0]);
  x = to_h<kBF16>(u.x);
  y = to_h<kBF16>(u.y);
}

// (Through L1: past it, one token costs 0.25 us more and 8192 tokens 0.9.)
__device__ __forceinline__ uint64_t position_at(const void* positions, int bits, int64_t i) {
  return bits == 64 ? static_cast<uint64_t>(static_cast<const long long*>(positions)[i])
                    : static_cast<uint64_t>(static_cast<int64_t>(static_cast<const int*>(positions)[i]));
}

// Where chunk c of a head lies: its two runs, and (after turn_to) the cosines and sines of its
// pairs for token (b, t); chunks past the pairs cover the elements that are copied.
template <int VEC, bool kAdj>
struct Chunk {
  int at0, at1;
  bool copied;
  float cs[VEC], sn[VEC];

  __device__ __forceinline__ Chunk(const fa4d_rotary_table& tab, int c) {
    const int pairs = tab.rotary_dim / 2, turned = pairs / VEC;
    copied = c >= turned;
    at0 = copied ? tab.rotary_dim + (c - turned) * 2 * VEC : (kAdj ? 2 * c * VEC : c * VEC);
    at1 = (kAdj || copied) ? at0 + VEC : pairs + c * VEC;
  }
  __device__ __forceinline__ void turn_to(const fa4d_rotary_table& tab, const void* positions, int bits,
                                          const int64_t (&ps)[3], int64_t b, int64_t t, int c, bool inverse) {
    if (copied) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = c * VEC + j;
      const uint64_t p = position_at(positions, bits, tab.axis[i] * ps[0] + b * ps[1] + t * ps[2]);
      // Nearest multiple of 2^-32 turns, as a signed fraction of half a turn.
      const int32_t frac = static_cast<int32_t>((p * tab.turn[i] + 0x80000000ull) >> 32);
      sincospif(static_cast<float>(frac) * 4.656612873077393e-10f, &sn[j], &cs[j]);  // 2^-31
      if (inverse) sn[j] = -sn[j];
    }
  }
};

}  // namespace fa4d
