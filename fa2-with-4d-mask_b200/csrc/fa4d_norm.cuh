// fa4d_norm.cuh — a head's elements over the lanes of a row, in fp32: the norm of the head and the
// turn by its position, for the kernels that normalise queries and keys.
#pragma once

#include "fa4d_rotary.cuh"

namespace fa4d {

// A row (one head of one token) lies over `lanes` neighbouring lanes of a warp, a power of two: with
// VEC = 8 each has a chunk of 8 pairs (lanes past the last chunk idle), with VEC = 1 all 32 have up
// to 4 chunks of one pair, 32 apart.
template <int VEC>
constexpr int kRowChunks = VEC == 1 ? 4 : 1;
template <int VEC>
constexpr int kRowPairs = VEC * kRowChunks<VEC>;  // of a lane

// Elements of pair j of chunk c of a row (past the pairs, of elements that are copied).  With VEC = 8
// a chunk is 8 elements of the first half of what is turned and 8 of the second, whichever the
// pairing, so that neighbouring lanes read neighbouring 16 bytes (with 32 bytes a lane, 16 at a time,
// every sector was asked for twice).
template <int VEC, bool kAdj>
struct PairAt {
  int e0, e1;
  __device__ __forceinline__ PairAt(const fa4d_rotary_table& tab, int c, int j) {
    const int pairs = tab.rotary_dim / 2, turned = pairs / VEC;
    const int at0 = c < turned ? c * (kAdj && VEC == 1 ? 2 : VEC) : tab.rotary_dim + (c - turned) * 2 * VEC;
    const int at1 = c < turned ? (kAdj && VEC == 1 ? at0 + 1 : pairs + c * VEC) : at0 + VEC;
    if (kAdj && VEC > 1) {
      e0 = j < VEC / 2 ? at0 + 2 * j : at1 + 2 * j - VEC;
      e1 = e0 + 1;
    } else {
      e0 = at0 + j;
      e1 = at1 + j;
    }
  }
};

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

// The sum over a row's lanes, in all of them; every lane of the warp takes part.  kLanes: known lanes
// of a row, or 0.
template <int kLanes = 0>
__device__ __forceinline__ float row_sum(float x, int lanes) {
  if constexpr (kLanes > 0) {
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  } else {
    for (int o = lanes / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  }
  return x;
}

__device__ __forceinline__ uint64_t minus(uint64_t x) { return x ^ 0x8000000080000000ull; }

// What a lane holds of a row: pair j is (a_j, b_j) (past the pairs, elements that are copied); two
// pairs beside one another lie packed, for the packed arithmetic.
template <int VEC>
struct Pairs {
  static constexpr int kTwo = kRowPairs<VEC> / 2;
  uint64_t a[kTwo], b[kTwo];

  __device__ __forceinline__ float squares() const {
    uint64_t s = f2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kTwo; ++j) s = ffma2(a[j], a[j], ffma2(b[j], b[j], s));
    const float2 t = f2_split(s);
    return t.x + t.y;
  }
  // Times w / sqrt(v), and into `low` what the roundings leave out.
  __device__ __forceinline__ void normalise(float v, const Pairs& w, Pairs& low) {
    const float r = rsqrtf(v), h = v * r;
    // One step of Newton's.  Squares beyond fp32 give r = 0, whose step would be 0 times infinity.
    const float e = fmaf(-h, r, 1.f) - fmaf(v, r, -h) * r, r_low = r > 0.f ? 0.5f * r * e : 0.f;
    const uint64_t rr = f2(r, r), rl = f2(r_low, r_low);
#pragma unroll
    for (int j = 0; j < kTwo; ++j) {
      auto one = [&](uint64_t& x, uint64_t weight, uint64_t& rest) {
        const uint64_t n = fmul2(x, rr), nl = ffma2(x, rl, ffma2(x, rr, minus(n)));
        const uint64_t y = fmul2(n, weight);
        rest = ffma2(nl, weight, ffma2(n, weight, minus(y)));
        x = y;
      };
      one(a[j], w.a[j], low.a[j]);
      one(b[j], w.b[j], low.b[j]);
    }
  }
  __device__ __forceinline__ void times(float r) {
    const uint64_t rr = f2(r, r);
#pragma unroll
    for (int j = 0; j < kTwo; ++j) {
      a[j] = fmul2(a[j], rr);
      b[j] = fmul2(b[j], rr);
    }
  }
};

// The raw elements of a lane's chunks, as they are loaded and stored.
template <int VEC>
struct Raw {
  typename Run<VEC>::T x[kRowChunks<VEC>], y[kRowChunks<VEC>];
};

// Cosines and sines of two angles, each in 2^-32 turns, packed: y, what is left beside the nearest
// quarter turn (at most 1/8, rounded to 24 bits), goes to polynomials in y^2, sin(2 pi y) = y S(y^2) and
// cos(2 pi y) = 1 + y^2 C(y^2), and the quarter swaps them and sets their signs.  The coefficients
// were fitted for this library (least squares on Chebyshev nodes, reweighted toward the minimax; 3e-9
// and 3e-10 off, with the coefficients rounded to fp32 2.4e-8 and 1.3e-8); with the arithmetic's
// rounding the results are off by at most 2^-23 (1.1e-7 over 2 million angles), and whole quarters are
// exact.  About 20 instructions an angle: with sincospif, whose argument has to hold whole half turns
// as well, angles were a third of what these kernels execute.
__device__ __forceinline__ void cos_sin2(uint32_t f0, uint32_t f1, uint64_t& c, uint64_t& s) {
  const uint32_t q0 = f0 + 0x20000000u, q1 = f1 + 0x20000000u;  // the nearest quarter in the top two bits
  const int32_t r0 = static_cast<int32_t>(f0 - (q0 & 0xC0000000u)), r1 = static_cast<int32_t>(f1 - (q1 & 0xC0000000u));
  auto both = [](float x) { return f2(x, x); };
  const uint64_t y = fmul2(f2(static_cast<float>(r0), static_cast<float>(r1)), both(2.3283064365386963e-10f));  // 2^-32
  const uint64_t u = fmul2(y, y);
  uint64_t S = ffma2(both(-75.40207f), u, both(81.59255f));
  S = fmul2(ffma2(ffma2(S, u, both(-41.341663f)), u, both(6.2831855f)), y);
  uint64_t C = ffma2(both(59.475986f), u, both(-85.4502f));
  C = ffma2(ffma2(ffma2(C, u, both(64.93938f)), u, both(-19.739208f)), u, both(1.f));
  const float2 si = f2_split(S), co = f2_split(C);
  auto place = [](uint32_t q, float si, float co, float& cq, float& sq) {
    const bool swap = q & 0x40000000u;
    sq = __uint_as_float(__float_as_uint(swap ? co : si) ^ (q & 0x80000000u));
    cq = __uint_as_float(__float_as_uint(swap ? si : co) ^ ((q + 0x40000000u) & 0x80000000u));
  };
  float c0, c1, s0, s1;
  place(q0, si.x, co.x, c0, s0);
  place(q1, si.y, co.y, c1, s1);
  c = f2(c0, c1);
  s = f2(s0, s1);
}

// The table's turns and axes in shared memory, laid so that the lanes of a row read neighbours (a
// kernel parameter is read one address at a time).
template <int VEC>
struct Turns {
  uint64_t turn[FA4D_ROTARY_MAX_PAIRS];
  uint8_t axis[FA4D_ROTARY_MAX_PAIRS];
  uint8_t several[FA4D_ROTARY_MAX_PAIRS / VEC];  // whether a chunk's pairs follow several axes
  static constexpr int kChunks = FA4D_ROTARY_MAX_PAIRS / VEC;
  static __device__ __forceinline__ int at(int chunk, int j) { return j * kChunks + chunk; }
  // All threads of the block; a barrier follows.
  template <bool kAdj>
  __device__ __forceinline__ void fill(const fa4d_rotary_table& tab) {
    for (int i = threadIdx.x; i < tab.rotary_dim / 2; i += blockDim.x) {
      const int c = i / VEC, j = i % VEC;
      auto pair = [&](int k) {
        const PairAt<VEC, kAdj> e(tab, c, k);
        return kAdj ? e.e0 / 2 : e.e0;
      };
      turn[at(c, j)] = tab.turn[pair(j)];
      axis[at(c, j)] = tab.axis[pair(j)];
      if (j == 0) {
        bool differ = false;
        for (int k = 1; k < VEC; ++k) differ = differ || tab.axis[pair(k)] != tab.axis[pair(0)];
        several[c] = differ;
      }
    }
  }
};

// A norm's weights in shared memory: of each chunk its pairs' first elements, then the second ones,
// four at a time, so that the lanes of a row read neighbours.  They stay there, since registers are
// what the kernels lack (and each lane reading its elements from memory took as many requests as
// eight heads' tokens).
template <int VEC>
struct Weights {
  static constexpr int kQuads = VEC == 1 ? 1 : VEC / 2;  // of a chunk (one pair: half of one)
  static constexpr int kChunks = FA4D_ROTARY_MAX_PAIRS / VEC;
  float4 w[kQuads * kChunks];
  // All threads of the block; a barrier follows.
  template <bool kBF16, bool kAdj>
  __device__ __forceinline__ void fill(const fa4d_rotary_table& tab, const void* from, bool f32) {
    for (int i = threadIdx.x; i < FA4D_ROTARY_MAX_PAIRS; i += blockDim.x) {
      const int c = i / VEC, j = i % VEC;
      if (i >= tab.D / 2) {  // lanes past the last chunk take part in sums
        set(c, j, 0.f);
        set(c, VEC + j, 0.f);
        continue;
      }
      const PairAt<VEC, kAdj> e(tab, c, j);
      auto get = [&](int e) {
        return f32 ? __ldcg(static_cast<const float*>(from) + e) : to_f<kBF16>(__ldcg(static_cast<const uint16_t*>(from) + e));
      };
      set(c, j, get(e.e0));
      set(c, VEC + j, get(e.e1));
    }
  }
  __device__ __forceinline__ void set(int c, int k, float x) {
    reinterpret_cast<float*>(&w[(k / 4) * kChunks + c])[k % 4] = x;
  }
  __device__ __forceinline__ float of(int c, int k) const { return reinterpret_cast<const float*>(&w[(k / 4) * kChunks + c])[k % 4]; }
};

// a A + b B, or a A where B is 0 (an infinite b and B = 0 make NaN).
__device__ __forceinline__ uint64_t mix_apart(uint64_t a, uint64_t A, uint64_t b, uint64_t B) {
  const float2 x = f2_split(a), u = f2_split(A), y = f2_split(b), v = f2_split(B);
  return f2(v.x == 0.f ? x.x * u.x : fmaf(x.x, u.x, y.x * v.x), v.y == 0.f ? x.y * u.y : fmaf(x.y, u.y, y.y * v.y));
}

// The cosines and sines of a lane's pairs.
template <int VEC>
struct Turn {
  uint64_t c[kRowPairs<VEC> / 2], s[kRowPairs<VEC> / 2];
  // Turned in place; `copied` as for back.
  __device__ __forceinline__ void on(Pairs<VEC>& p, bool copied) const {
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      const uint64_t a = p.a[j], b = p.b[j];
      if (copied) {
        p.a[j] = mix_apart(a, c[j], b, minus(s[j]));
        p.b[j] = mix_apart(b, c[j], a, s[j]);
      } else {
        p.a[j] = ffma2(a, c[j], fmul2(b, minus(s[j])));
        p.b[j] = ffma2(b, c[j], fmul2(a, s[j]));
      }
    }
  }
  // Turned in place with what roundings left out of p so far (`low`) and of the turn's first products.
  __device__ __forceinline__ void on_exact(Pairs<VEC>& p, const Pairs<VEC>& low, bool copied) const {
    if (copied) {  // (a chunk of them is not turned, or single pairs are)
      on(p, true);
      return;
    }
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      const uint64_t a = p.a[j], b = p.b[j], m = minus(s[j]);
      const uint64_t u = fmul2(b, m), v = fmul2(a, s[j]);
      const uint64_t lu = ffma2(low.b[j], m, ffma2(low.a[j], c[j], ffma2(b, m, minus(u))));
      const uint64_t lv = ffma2(low.a[j], s[j], ffma2(low.b[j], c[j], ffma2(a, s[j], minus(v))));
      p.a[j] = fadd2(ffma2(a, c[j], u), lu);
      p.b[j] = fadd2(ffma2(b, c[j], v), lv);
    }
  }
  // Turned back.  `copied`: pairs with sine 0 are not to be mixed (see RowLane::copied).
  __device__ __forceinline__ void back(const Pairs<VEC>& d, Pairs<VEC>& g, bool copied) const {
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      if (copied) {
        g.a[j] = mix_apart(d.a[j], c[j], d.b[j], s[j]);
        g.b[j] = mix_apart(d.b[j], c[j], d.a[j], minus(s[j]));
      } else {
        g.a[j] = ffma2(d.a[j], c[j], fmul2(d.b[j], s[j]));
        g.b[j] = ffma2(d.b[j], c[j], fmul2(d.a[j], minus(s[j])));
      }
    }
  }
};

// The turn with a norm's weights: (a, b) becomes (a A + b B, b C + a E).
template <int VEC>
struct Factors {
  uint64_t A[kRowPairs<VEC> / 2], B[kRowPairs<VEC> / 2], C[kRowPairs<VEC> / 2], E[kRowPairs<VEC> / 2];
  __device__ __forceinline__ void set(const Turn<VEC>& t) {
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      A[j] = C[j] = t.c[j];
      B[j] = minus(t.s[j]);
      E[j] = t.s[j];
    }
  }
  __device__ __forceinline__ void weigh(const Pairs<VEC>& w) {
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      A[j] = fmul2(w.a[j], A[j]);
      B[j] = fmul2(w.b[j], B[j]);
      C[j] = fmul2(w.b[j], C[j]);
      E[j] = fmul2(w.a[j], E[j]);
    }
  }
  // `copied`: as for Turn::back.
  __device__ __forceinline__ void turn(Pairs<VEC>& p, bool copied) const {
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) {
      const uint64_t a = p.a[j], b = p.b[j];
      if (copied) {
        p.a[j] = mix_apart(a, A[j], b, B[j]);
        p.b[j] = mix_apart(b, C[j], a, E[j]);
      } else {
        p.a[j] = ffma2(a, A[j], fmul2(b, B[j]));
        p.b[j] = ffma2(b, C[j], fmul2(a, E[j]));
      }
    }
  }
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
      at0[i] = PairAt<VEC, kAdj>(tab, c, 0).e0;
      at1[i] = kAdj && VEC > 1 ? PairAt<VEC, kAdj>(tab, c, VEC / 2).e0 : PairAt<VEC, kAdj>(tab, c, 0).e1;
      if (c < chunks) {
        live |= 1u << i;
        if (c < tab.rotary_dim / 2 / VEC) turned |= 1u << i;
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
  // This lane's elements of a norm's weights.
  __device__ __forceinline__ void weights(const Weights<VEC>& w, int lane, Pairs<VEC>& p) const {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const bool u = (live >> i) & 1u, v = (live >> (i + 1)) & 1u;
        p.a[i / 2] = f2(u ? w.of(lane + 32 * i, 0) : 0.f, v ? w.of(lane + 32 * i + 32, 0) : 0.f);
        p.b[i / 2] = f2(u ? w.of(lane + 32 * i, 1) : 0.f, v ? w.of(lane + 32 * i + 32, 1) : 0.f);
      }
    } else {
#pragma unroll
      for (int q = 0; q < VEC / 4; ++q) {
        const float4 x = w.w[q * Weights<VEC>::kChunks + lane], y = w.w[(VEC / 4 + q) * Weights<VEC>::kChunks + lane];
        p.a[2 * q] = f2(x.x, x.y), p.a[2 * q + 1] = f2(x.z, x.w);
        p.b[2 * q] = f2(y.x, y.y), p.b[2 * q + 1] = f2(y.z, y.w);
      }
    }
  }
  // The cosines and sines of the row's pairs at token (b, t).
  __device__ __forceinline__ void angles(const Turns<VEC>& turns, const void* positions, int bits, const int64_t (&ps)[3],
                                         int64_t b, int64_t t, int lane, Turn<VEC>& out) const {
    uint32_t f[kRowPairs<VEC>];  // nearest multiples of 2^-32 turns
#pragma unroll
    for (int i = 0; i < kRowChunks<VEC>; ++i)
      if ((turned >> i) & 1u) {
        const int64_t here = b * ps[1] + t * ps[2];
        const int c = lane + 32 * i;
        const uint64_t first = position_at(positions, bits, turns.axis[turns.at(c, 0)] * ps[0] + here);
        const bool several = turns.several[c];  // mostly a chunk follows one axis
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int at = turns.at(c, j);
          uint64_t p = first;
          if (several) p = position_at(positions, bits, turns.axis[at] * ps[0] + here);
          f[VEC * i + j] = static_cast<uint32_t>((p * turns.turn[at] + 0x80000000ull) >> 32);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[VEC * i + j] = 0;  // cosine 1 and sine 0, exactly
      }
#pragma unroll
    for (int j = 0; j < kRowPairs<VEC> / 2; ++j) cos_sin2(f[2 * j], f[2 * j + 1], out.c[j], out.s[j]);
  }
  // Chunks that are copied keep apart what the turn would mix: 0 * infinity is not a number.
  __device__ __forceinline__ bool copied() const { return turned != live; }
};

template <bool kBF16, bool kAdj, int VEC>
__device__ __forceinline__ void unpack_pairs(const Raw<VEC>& r, Pairs<VEC>& p) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      p.a[i / 2] = f2(to_f<kBF16>(r.x[i]), to_f<kBF16>(r.x[i + 1]));
      p.b[i / 2] = f2(to_f<kBF16>(r.y[i]), to_f<kBF16>(r.y[i + 1]));
    }
  } else {
    constexpr int W = VEC / 2;  // words of a run
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&r.x[0]);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&r.y[0]);
    if constexpr (kAdj) {
#pragma unroll
      for (int w = 0; w < W; w += 2) {
        const float2 u = unpack2<kBF16>(x[w]), v = unpack2<kBF16>(x[w + 1]), s = unpack2<kBF16>(y[w]), t = unpack2<kBF16>(y[w + 1]);
        p.a[w / 2] = f2(u.x, v.x), p.b[w / 2] = f2(u.y, v.y);
        p.a[(w + W) / 2] = f2(s.x, t.x), p.b[(w + W) / 2] = f2(s.y, t.y);
      }
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 u = unpack2<kBF16>(x[w]), v = unpack2<kBF16>(y[w]);
        p.a[w] = f2(u.x, u.y);
        p.b[w] = f2(v.x, v.y);
      }
    }
  }
}
template <bool kBF16, bool kAdj, int VEC>
__device__ __forceinline__ void pack_pairs(const Pairs<VEC>& p, Raw<VEC>& r) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 a = f2_split(p.a[i / 2]), b = f2_split(p.b[i / 2]);
      r.x[i] = to_h<kBF16>(a.x), r.x[i + 1] = to_h<kBF16>(a.y);
      r.y[i] = to_h<kBF16>(b.x), r.y[i + 1] = to_h<kBF16>(b.y);
    }
  } else {
    constexpr int W = VEC / 2;
    uint32_t* x = reinterpret_cast<uint32_t*>(&r.x[0]);
    uint32_t* y = reinterpret_cast<uint32_t*>(&r.y[0]);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float2 a = f2_split(p.a[j]), b = f2_split(p.b[j]);
      if constexpr (kAdj) {
        uint32_t* z = j < W / 2 ? x + 2 * j : y + 2 * j - W;
        z[0] = pack2<kBF16>(a.x, b.x);
        z[1] = pack2<kBF16>(a.y, b.y);
      } else {
        x[j] = pack2<kBF16>(a.x, a.y);
        y[j] = pack2<kBF16>(b.x, b.y);
      }
    }
  }
}

// The heads [first, end) of a token, normalised (weights; null: not) and turned.
// kHeads rows' loads are in flight together.
template <bool kBF16, bool kAdj, int VEC, int kHeads>
__device__ __forceinline__ void norm_heads(const fa4d_rotary_table& tab, const Turns<VEC>& turns, const RowLane<VEC, kAdj>& at, const Weights<VEC>* weights,
                                           float eps, int lanes, int lane, bool live, const uint16_t* src, int64_t src_head,
                                           uint16_t* dst, int64_t dst_head, int first, int end, const void* positions, int bits,
                                           const int64_t (&ps)[3], int64_t b, int64_t t) {
  Factors<VEC> factors;
  const bool copied = at.copied();
  for (int h0 = first; h0 < end; h0 += kHeads) {
    Raw<VEC> raw[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u)
      if (live && h0 + u < end) at.load(src + (h0 + u) * src_head, raw[u]);
    // The angles, while the first heads are on their way.
    if (h0 == first && live) {
      Turn<VEC> turn;
      at.angles(turns, positions, bits, ps, b, t, lane, turn);
      factors.set(turn);
      if (weights) {
        Pairs<VEC> w;
        at.weights(*weights, lane, w);
        factors.weigh(w);
      }
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      Pairs<VEC> p;
      unpack_pairs<kBF16, kAdj>(raw[u], p);
      if (weights) p.times(rsqrtf(row_sum(p.squares(), lanes) * (1.f / tab.D) + eps));
      if (!live || h0 + u >= end) continue;
      factors.turn(p, copied);
      pack_pairs<kBF16, kAdj>(p, raw[u]);
      at.store(dst + (h0 + u) * dst_head, raw[u]);
    }
  }
}

}  // namespace fa4d
