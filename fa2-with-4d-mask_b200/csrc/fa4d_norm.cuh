// fa4d_norm.cuh — a head's elements over the lanes of a row, in fp32: the norm of the head and the
// turn by its position, for the kernels that normalise queries and keys.
#pragma once

#include "fa4d_rotary.cuh"

namespace fa4d {

// A row (one head of one token) lies over `lanes` neighbouring lanes of a warp, a power of two: with
// VEC = 8 each has a chunk of 8 pairs (lanes past the last chunk idle), with VEC = 1 all 32 have up
// to 4 chunks of one pair, 32 apart.
template <int VEC>
constexpr int kRowChunks = VEC == 8 ? 1 : 4;
template <int VEC>
constexpr int kRowPairs = VEC * kRowChunks<VEC>;  // of a lane

inline int chunks_of(const fa4d_rotary_table& tab, int vec) {
  return tab.rotary_dim / 2 / vec + (tab.D - tab.rotary_dim) / (2 * vec);
}
// Lanes of a row.
inline int row_lanes(const fa4d_rotary_table& tab, int vec) {
  if (vec == 1) return 32;
  int lanes = 1;
  while (lanes < chunks_of(tab, vec)) lanes *= 2;
  return lanes;
}

// The sum over a row's lanes, in all of them; every lane of the warp takes part.
__device__ __forceinline__ float row_sum(float x, int lanes) {
  for (int o = lanes / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// What a lane holds of a row: pair j is (a[j], b[j]) (past the pairs, elements that are copied).
template <int VEC>
struct Pairs {
  float a[kRowPairs<VEC>], b[kRowPairs<VEC>];

  __device__ __forceinline__ float squares() const {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC>; ++j) s = fmaf(a[j], a[j], fmaf(b[j], b[j], s));
    return s;
  }
};

// The raw elements of a lane's chunks, as they are loaded and stored.
template <int VEC>
struct Raw {
  typename Run<VEC>::T x[kRowChunks<VEC>], y[kRowChunks<VEC>];
};

// A lane's place in its row.
template <int VEC, bool kAdj>
struct RowLane {
  int at0[kRowChunks<VEC>], at1[kRowChunks<VEC>];
  uint32_t live, turned;  // bit i: chunk i exists, and its pairs turn

  __device__ __forceinline__ RowLane(const fa4d_rotary_table& tab, int lane, int chunks) : live(0), turned(0) {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i) {
      const int c = lane + 32 * i;
      const Chunk<VEC, kAdj> ch(tab, c);
      at0[i] = ch.at0;
      at1[i] = ch.at1;
      if (c < chunks) {
        live |= 1u << i;
        if (!ch.copied) turned |= 1u << i;
      }
    }
  }
  __device__ __forceinline__ void load(const uint16_t* row, Raw<VEC>& r) const {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
      if ((live >> i) & 1u) {
        r.x[i] = Run<VEC>::load(row + at0[i]);
        r.y[i] = Run<VEC>::load(row + at1[i]);
      } else {
        r.x[i] = r.y[i] = {};
      }
  }
  __device__ __forceinline__ void store(uint16_t* row, const Raw<VEC>& r) const {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
      if ((live >> i) & 1u) {
        Run<VEC>::store(row + at0[i], r.x[i]);
        Run<VEC>::store(row + at1[i], r.y[i]);
      }
  }
  // A vector of D elements (a norm's weights), fp32 or 16-bit.
  template <bool kBF16>
  __device__ __forceinline__ void vector(const void* w, bool f32, Pairs<VEC>& p) const {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool ok = (live >> i) & 1u;
        const int e0 = kAdj && VEC == 8 ? at0[i] + 2 * j : at0[i] + j, e1 = kAdj && VEC == 8 ? e0 + 1 : at1[i] + j;
        auto at = [&](int e) {
          if (!ok) return 0.f;
          return f32 ? __ldcg(static_cast<const float*>(w) + e) : to_f<kBF16>(__ldcg(static_cast<const uint16_t*>(w) + e));
        };
        p.a[VEC * i + j] = at(e0);
        p.b[VEC * i + j] = at(e1);
      }
  }
  // The cosines and sines of the row's pairs at token (b, t).
  __device__ __forceinline__ void angles(const fa4d_rotary_table& tab, const void* positions, int bits,
                                         const int64_t (&ps)[3], int64_t b, int64_t t, int lane,
                                         float (&cs)[kRowPairs<VEC>], float (&sn)[kRowPairs<VEC>]) const {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
      if ((turned >> i) & 1u) {
        Chunk<VEC, kAdj> ch(tab, lane + 32 * i);
        ch.turn_to(tab, positions, bits, ps, b, t, lane + 32 * i, false);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          cs[VEC * i + j] = ch.cs[j];
          sn[VEC * i + j] = ch.sn[j];
        }
      }
  }
  // Turned by the angles (sign 1) or back (sign -1).
  __device__ __forceinline__ void turn(Pairs<VEC>& p, const float (&cs)[kRowPairs<VEC>], const float (&sn)[kRowPairs<VEC>],
                                       float sign) const {
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
      if ((turned >> i) & 1u) {
#pragma unroll
        for (int j = VEC * i; j < VEC * (i + 1); ++j) {
          const float2 u = turned_pair(p.a[j], p.b[j], cs[j], sign * sn[j]);
          p.a[j] = u.x;
          p.b[j] = u.y;
        }
      }
  }
  static __device__ __forceinline__ float2 turned_pair(float a, float b, float c, float s) { return fa4d::turned(a, b, c, s); }
};

template <bool kBF16, bool kAdj>
__device__ __forceinline__ void unpack_pairs(const Raw<8>& r, Pairs<8>& p) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(&r.x[0]);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(&r.y[0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 u = unpack2<kBF16>(x[w]), v = unpack2<kBF16>(y[w]);
    if (kAdj) {
      p.a[w] = u.x, p.b[w] = u.y;
      p.a[w + 4] = v.x, p.b[w + 4] = v.y;
    } else {
      p.a[2 * w] = u.x, p.a[2 * w + 1] = u.y;
      p.b[2 * w] = v.x, p.b[2 * w + 1] = v.y;
    }
  }
}
template <bool kBF16, bool kAdj>
__device__ __forceinline__ void unpack_pairs(const Raw<1>& r, Pairs<1>& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p.a[i] = to_f<kBF16>(r.x[i]);
    p.b[i] = to_f<kBF16>(r.y[i]);
  }
}
template <bool kBF16, bool kAdj>
__device__ __forceinline__ void pack_pairs(const Pairs<8>& p, Raw<8>& r) {
  uint32_t* x = reinterpret_cast<uint32_t*>(&r.x[0]);
  uint32_t* y = reinterpret_cast<uint32_t*>(&r.y[0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    x[w] = kAdj ? pack2<kBF16>(p.a[w], p.b[w]) : pack2<kBF16>(p.a[2 * w], p.a[2 * w + 1]);
    y[w] = kAdj ? pack2<kBF16>(p.a[w + 4], p.b[w + 4]) : pack2<kBF16>(p.b[2 * w], p.b[2 * w + 1]);
  }
}
template <bool kBF16, bool kAdj>
__device__ __forceinline__ void pack_pairs(const Pairs<1>& p, Raw<1>& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.x[i] = to_h<kBF16>(p.a[i]);
    r.y[i] = to_h<kBF16>(p.b[i]);
  }
}

// The heads [first, end) of a token, normalised (w; null: not) and turned.
// kHeads rows' loads are in flight together.
template <bool kBF16, bool kAdj, int VEC, int kHeads>
__device__ __forceinline__ void norm_heads(const fa4d_rotary_table& tab, const RowLane<VEC, kAdj>& at, const Pairs<VEC>* w,
                                           float eps, int lanes, int lane, bool live, const uint16_t* src, int64_t src_head,
                                           uint16_t* dst, int64_t dst_head, int first, int end, const void* positions, int bits,
                                           const int64_t (&ps)[3], int64_t b, int64_t t) {
  float cs[kRowPairs<VEC>], sn[kRowPairs<VEC>];
  for (int h0 = first; h0 < end; h0 += kHeads) {
    Raw<VEC> raw[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u)
      if (live && h0 + u < end) at.load(src + (h0 + u) * src_head, raw[u]);
    // The angles, while the first heads are on their way.
    if (h0 == first && live) at.angles(tab, positions, bits, ps, b, t, lane, cs, sn);
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      Pairs<VEC> p;
      unpack_pairs<kBF16, kAdj>(raw[u], p);
      if (w) {
        const float r = rsqrtf(row_sum(p.squares(), lanes) * (1.f / tab.D) + eps);
#pragma unroll
        for (int j = 0; j < kRowPairs<VEC>; ++j) {
          p.a[j] = p.a[j] * r * w->a[j];
          p.b[j] = p.b[j] * r * w->b[j];
        }
      }
      if (!live || h0 + u >= end) continue;
      at.turn(p, cs, sn, 1.f);
      pack_pairs<kBF16, kAdj>(p, raw[u]);
      at.store(dst + (h0 + u) * dst_head, raw[u]);
    }
  }
}

}  // namespace fa4d
