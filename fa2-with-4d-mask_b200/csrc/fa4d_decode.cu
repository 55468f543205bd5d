// fa4d_decode.cu — attention of a few new tokens over long caches: the keys are divided over
// all warps of the GPU (decode_kernel), and the partial results joined (join_kernel).
//
// o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m), x_j = scale log2(e) q.k_j: numerator and
// denominator over any set of keys, each with its own m, are joined exactly by factors
// 2^(m - m_all).
#include "fa4d.h"
#include "fa4d_decode.h"
#include "fa4d_ptx.cuh"

namespace fa4d {

namespace {

constexpr float kNegInf = -INFINITY;

template <int D>
struct DecodeShape {
  // Bytes of a key's row in shared memory: a power of two, so that the 16-byte chunks of
  // eight rows, each stored at (chunk ^ row % 8), lie in different banks.
  static constexpr int kPitch = D == 96 ? 256 : 2 * D;
  static constexpr int kTile = kUnitKeys * kPitch;  // K or V of a unit
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kBytes = kDecodeWarps * kStages * kStage;
  static constexpr int kCtas = D == 256 ? 1 : 2;  // on an SM
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c (16 x 8, fp32) += a (16 x 16) b (16 x 8)
template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ int length_of(const DecodeParams& p, int b) { return min(max(__ldg(p.lengths + b), 0), p.C); }
__device__ __forceinline__ int units_of(int keys) { return (keys + kUnitKeys - 1) / kUnitKeys; }

// Units of the requests before b (all of them for b = B), per KV head and row tile.
__device__ __forceinline__ int64_t units_before(const DecodeParams& p, int b, int lane) {
  int64_t n = 0;
  for (int i = lane; i < b; i += 32) n += units_of(length_of(p, i));
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// Units of a warp, from the number of units in all.
__device__ __forceinline__ int64_t share_of(const DecodeParams& p, int64_t total) {
  return max(static_cast<int64_t>(p.min_units), (total + p.warps - 1) / p.warps);
}

// A place on the line of units.
struct Place {
  bool prefix;
  int b, hk, tile;  // the item (b unused in the prefix)
  int u, units;     // unit within the item, units of the item
  int keys;         // keys of the item

  __device__ __forceinline__ int item(const DecodeParams& p) const {
    return prefix ? hk * p.prefix_tiles + tile : (p.prefix_tiles + b * p.tiles) * p.Hk + hk * p.tiles + tile;
  }
  // First request at or after b that has keys (B: none).
  __device__ __forceinline__ void to_request(const DecodeParams& p, int from) {
    prefix = false;
    u = hk = tile = 0;
    keys = units = 0;
    for (b = from; b < p.B; ++b) {
      keys = length_of(p, b);
      units = units_of(keys);
      if (units) break;
    }
  }
  // To the next unit; true if it is of another item.
  __device__ __forceinline__ bool advance(const DecodeParams& p) {
    if (++u < units) return false;
    u = 0;
    if (++tile < (prefix ? p.prefix_tiles : p.tiles)) return true;
    tile = 0;
    if (++hk < p.Hk) return true;
    to_request(p, prefix ? 0 : b + 1);
    return true;
  }
};

// The place of unit `at` (which exists).
__device__ __forceinline__ Place find_place(const DecodeParams& p, int64_t at, int lane) {
  Place w;
  const int64_t prefix_all = static_cast<int64_t>(p.prefix_tiles) * p.Hk * p.prefix_units;
  if (at < prefix_all) {
    const int64_t item = at / p.prefix_units;
    w.prefix = true;
    w.b = 0;
    w.hk = static_cast<int>(item / p.prefix_tiles);
    w.tile = static_cast<int>(item - static_cast<int64_t>(w.hk) * p.prefix_tiles);
    w.u = static_cast<int>(at - item * p.prefix_units);
    w.units = p.prefix_units;
    w.keys = p.P;
    return w;
  }
  at -= prefix_all;
  const int64_t each = static_cast<int64_t>(p.Hk) * p.tiles;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    const int mine = b < p.B ? units_of(length_of(p, b)) : 0;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t left = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += left;
    }
    const unsigned past = __ballot_sync(0xffffffffu, upto * each > at);
    if (past) {
      const int l = __ffs(past) - 1;
      at -= (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, mine, l)) * each;
      w.prefix = false;
      w.b = b0 + l;
      w.keys = length_of(p, w.b);
      w.units = units_of(w.keys);
      const int64_t item = at / w.units;
      w.hk = static_cast<int>(item / p.tiles);
      w.tile = static_cast<int>(item - static_cast<int64_t>(w.hk) * p.tiles);
      w.u = static_cast<int>(at - item * w.units);
      return w;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31) * each;
  }
  w.to_request(p, p.B);
  return w;
}

// One warp: its units in order, each 16 keys of K and V brought by cp.async into the warp's
// own ring (no barrier between warps), x = Q K^T and P V by m16n8k16 products with the
// fp32 output row tile in registers.  Memory-bound: a row tile of 16 needs 16 FLOP per byte
// of K and V.
template <int D, bool kBF16, bool kMask>
__global__ void __launch_bounds__(32 * kDecodeWarps, DecodeShape<D>::kCtas) decode_kernel(
    const __grid_constant__ DecodeParams p) {
  using S = DecodeShape<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * kDecodeWarps + (threadIdx.x >> 5);
  pdl_launch();

  const int64_t total = static_cast<int64_t>(p.prefix_tiles) * p.Hk * p.prefix_units +
                        units_before(p, p.B, lane) * p.Hk * p.tiles;
  const int64_t share = share_of(p, total);
  const int64_t first = warp * share;
  const int n = static_cast<int>(max(min(share, total - first), static_cast<int64_t>(0)));
  if (n > 0) {
    const uint32_t ring = smem_u32(smem) + (threadIdx.x >> 5) * S::kStages * S::kStage;
    Place in = find_place(p, first, lane);
    Place at = in;

    // K and V of the unit at `in` into a stage; rows past the item's keys are zeros.
    auto bring = [&](int stage) {
      const int64_t ks = in.prefix ? p.pk_stride[0] : p.k_stride[1], vs = in.prefix ? p.pv_stride[0] : p.v_stride[1];
      const uint16_t* kb = in.prefix ? static_cast<const uint16_t*>(p.pk) + in.hk * p.pk_stride[1]
                                     : static_cast<const uint16_t*>(p.k) + in.b * p.k_stride[0] + in.hk * p.k_stride[2];
      const uint16_t* vb = in.prefix ? static_cast<const uint16_t*>(p.pv) + in.hk * p.pv_stride[1]
                                     : static_cast<const uint16_t*>(p.v) + in.b * p.v_stride[0] + in.hk * p.v_stride[2];
      const int key0 = in.u * kUnitKeys;
      const uint32_t base = ring + stage * S::kStage;
      constexpr int kChunks = D / 8;
#pragma unroll
      for (int i = 0; i < kUnitKeys * kChunks / 32; ++i) {
        const int id = i * 32 + lane, row = id / kChunks, c = id - row * kChunks;
        const bool valid = key0 + row < in.keys;
        const int64_t key = valid ? key0 + row : key0;
        const uint32_t dst = base + row * S::kPitch + ((c ^ (row & 7)) << 4);
        cp_async16(dst, kb + key * ks + c * 8, valid);
        cp_async16(dst + S::kTile, vb + key * vs + c * 8, valid);
      }
    };

    int brought = 0;
    auto bring_next = [&]() {
      if (brought < n) {
        bring(brought % S::kStages);
        ++brought;
        if (brought < n) in.advance(p);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) bring_next();

    uint32_t qf[D / 16][4];
    float acc[D / 8][4];
    float m[2], l[2];
    int lim[2];              // keys below lim[i] are seen by row i of this thread
    const uint8_t* mrow[2];  // its mask row
    float* lrow[2];          // its row of logits, null where there is none
    const int col = 2 * (lane & 3);

    auto begin_item = [&]() {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = at.tile * 16 + (lane >> 2) + 8 * i;
        int64_t b = at.b, t = r / p.G;
        const int h = at.hk * p.G + r % p.G;
        bool valid = r < p.R;
        if (at.prefix) {
          b = t / p.T;
          t -= b * p.T;
          valid = b < p.B;
        }
        lim[i] = !valid ? 0 : at.prefix ? p.P : p.causal ? static_cast<int>(at.keys - p.T + t + 1) : at.keys;
        mrow[i] = nullptr;
        lrow[i] = nullptr;
        if (valid && !at.prefix) {
          if (kMask) mrow[i] = p.mask + b * p.mask_stride[0] + h * p.mask_stride[1] + t * p.mask_stride[2];
          if (p.logits) lrow[i] = p.logits + ((b * p.Hk + at.hk) * p.R + r) * p.logits_ld;
        }
        const uint16_t* row =
            static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2] + col;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[kk][i] = valid ? __ldg(reinterpret_cast<const uint32_t*>(row + 16 * kk)) : 0u;
          qf[kk][i + 2] = valid ? __ldg(reinterpret_cast<const uint32_t*>(row + 16 * kk + 8)) : 0u;
        }
        m[i] = kNegInf;
        l[i] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][e] = 0.f;
    };

    auto end_item = [&]() {
      const int64_t seg = warp + at.item(p);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = (lane >> 2) + 8 * i;
        if (r >= p.seg_rows) continue;
        const int64_t row = seg * p.seg_rows + r;
        if ((lane & 3) == 0) p.seg_ml[row] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<float2*>(p.seg_o + row * D + 8 * c + col) = make_float2(acc[c][2 * i], acc[c][2 * i + 1]);
      }
    };

    begin_item();
    for (int it = 0; it < n; ++it) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();
      bring_next();  // into the stage of the unit before this one
      const uint32_t sk = ring + (it % S::kStages) * S::kStage, sv = sk + S::kTile;

      float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(sk + row * S::kPitch + (((2 * kk + half) ^ (row & 7)) << 4), kf);
          mma16816<kBF16>(x[0], qf[kk], kf[0], kf[1]);
          mma16816<kBF16>(x[1], qf[kk], kf[2], kf[3]);
        }
      }
      // Scaled to log2 units; -inf where the row does not see the key.
      const int key0 = at.u * kUnitKeys;
      unsigned dead = 0xffffu;  // keys no row sees
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = e >> 1, kj = 8 * nt + col + (e & 1), j = key0 + kj;
          bool keep = j < lim[i];
          if (kMask && keep && mrow[i]) keep = mrow[i][j] != 0;
          x[nt][e] = keep ? x[nt][e] * p.scale_log2 : kNegInf;
          if (keep) dead &= ~(1u << kj);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lrow[i])
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
            if (key0 + 8 * nt + col < at.keys)
              *reinterpret_cast<float2*>(lrow[i] + key0 + 8 * nt + col) = make_float2(x[nt][2 * i], x[nt][2 * i + 1]);

      // A key that no row sees may hold anything: its V is cleared, since 0 * NaN is NaN.
      dead = __reduce_and_sync(0xffffffffu, dead);
      if (dead) {
        constexpr int kChunks = D / 8;
#pragma unroll 1
        for (int id = lane; id < kUnitKeys * kChunks; id += 32) {
          const int row = id / kChunks, c = id - row * kChunks;
          if ((dead >> row) & 1)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + row * S::kPitch + ((c ^ (row & 7)) << 4)),
                         "r"(0)
                         : "memory");
        }
        __syncwarp();
      }

      // Running maximum per row; the output is rescaled only where a maximum grew.
      float factor[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx, m[i]);
        factor[i] = m[i] == mx ? 1.f : ex2(m[i] - mx);
        m[i] = mx;
      }
      if (__any_sync(0xffffffffu, factor[0] != 1.f || factor[1] != 1.f)) {
        l[0] *= factor[0];
        l[1] *= factor[1];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          acc[c][0] *= factor[0];
          acc[c][1] *= factor[0];
          acc[c][2] *= factor[1];
          acc[c][3] *= factor[1];
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float sub = m[i] == kNegInf ? 0.f : m[i];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float p0 = ex2(x[nt][2 * i] - sub), p1 = ex2(x[nt][2 * i + 1] - sub);
          l[i] += p0 + p1;
          pf[2 * nt + i] = pack2<kBF16>(p0, p1);  // rounded to the type of V, as the product takes it
        }
      }
      {
        const int row = lane & 15, half = lane >> 4;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t vf[4];
          ldsm4_t(sv + row * S::kPitch + (((2 * c + half) ^ (row & 7)) << 4), vf);
          mma16816<kBF16>(acc[2 * c], pf, vf[0], vf[1]);
          mma16816<kBF16>(acc[2 * c + 1], pf, vf[2], vf[3]);
        }
      }
      if (at.u + 1 == at.units || it + 1 == n) end_item();
      if (it + 1 < n && at.advance(p)) begin_item();
    }
    cp_async_wait<0>();
  }
  // The join may start once this grid is through; it must then also find what the prefix
  // kernel before this one wrote.
  pdl_wait();
}

// ------------------------------------------------------------------ join

// Where the partial results of a row lie: `n` of them, the i-th at row first + i * step.
struct Parts {
  const float* o;
  const float2* ml;
  int64_t first, step;
  int n;
};

template <int D>
struct RowAcc {
  static constexpr int kEach = D / 32;  // elements of a lane: consecutive
  float v[kEach];
};

template <int D>
__device__ __forceinline__ void load_row(const float* row, int lane, float (&v)[D / 32]) {
  if constexpr (D == 64) {
    const float2 a = *reinterpret_cast<const float2*>(row + 2 * lane);
    v[0] = a.x, v[1] = a.y;
  } else if constexpr (D == 96) {
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = row[3 * lane + i];
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(row + (D / 32) * lane + 4 * i);
      v[4 * i] = a.x, v[4 * i + 1] = a.y, v[4 * i + 2] = a.z, v[4 * i + 3] = a.w;
    }
  }
}

constexpr int kJoinThreads = 128;
constexpr int kJoinKeys = 4 * kJoinThreads;  // own keys of a block that adds weights

// Blocks x < row_blocks join the output, a warp a row; the others add the weights of
// kJoinKeys own keys.
template <int D, bool kBF16>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ DecodeParams p, int row_blocks) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int hk = blockIdx.y, b = blockIdx.z;
  const bool adds = static_cast<int>(blockIdx.x) >= row_blocks;
  const int keys = length_of(p, b);
  const int key0 = (static_cast<int>(blockIdx.x) - row_blocks) * kJoinKeys;
  if (adds && key0 >= keys) return;

  const int64_t prefix_all = static_cast<int64_t>(p.prefix_tiles) * p.Hk * p.prefix_units;
  const int64_t each = static_cast<int64_t>(p.Hk) * p.tiles;
  const int64_t share = share_of(p, prefix_all + units_before(p, p.B, lane) * each);
  const int units = units_of(keys);
  const int64_t first_unit = prefix_all + units_before(p, b, lane) * each;
  pdl_wait();

  // The parts of row r: of its own keys, and of the prefix.
  auto parts_of_units = [&](int64_t from, int count, int64_t item, int row) {
    Parts x{p.seg_o, p.seg_ml, 0, p.seg_rows, 0};
    if (count > 0) {
      const int64_t w0 = from / share;
      x.n = static_cast<int>((from + count - 1) / share - w0 + 1);
      x.first = (w0 + item) * p.seg_rows + row;
    }
    return x;
  };
  auto own_parts = [&](int r) {
    const int64_t i = static_cast<int64_t>(hk) * p.tiles + r / 16;
    return parts_of_units(first_unit + i * units, units, static_cast<int64_t>(p.prefix_tiles) * p.Hk + b * each + i, r % 16);
  };
  auto prefix_parts = [&](int r) {
    const int64_t row = static_cast<int64_t>(b) * p.R + r;
    if (p.splits) {
      return Parts{p.pre_o, p.pre_ml, static_cast<int64_t>(hk) * p.splits * p.pre_rows + row, p.pre_rows, p.splits};
    }
    const int64_t i = static_cast<int64_t>(hk) * p.prefix_tiles + row / 16;
    return parts_of_units(i * p.prefix_units, p.prefix_tiles ? p.prefix_units : 0, i, static_cast<int>(row % 16));
  };
  // Maximum and sum over all parts of a row.
  auto total_of = [&](const Parts& x, const Parts& y) {
    float m = kNegInf, l = 0.f;
    for (int i = lane; i < x.n + y.n; i += 32) {
      const float2 ml = i < x.n ? x.ml[x.first + i * x.step] : y.ml[y.first + (i - x.n) * y.step];
      const float mx = fmaxf(m, ml.x);
      if (mx != kNegInf) l = l * ex2(m - mx) + ml.y * ex2(ml.x - mx);
      m = mx;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
      const float mx = fmaxf(m, m2);
      if (mx != kNegInf) l = l * ex2(m - mx) + l2 * ex2(m2 - mx);
      m = mx;
    }
    return make_float2(m, l);
  };

  if (!adds) {
    const int r = blockIdx.x * (kJoinThreads / 32) + wid;
    if (r >= p.R) return;
    const Parts x = prefix_parts(r), y = own_parts(r);
    const float2 all = total_of(x, y);
    float acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
    auto add = [&](const Parts& z) {
#pragma unroll 4
      for (int i = 0; i < z.n; ++i) {
        const int64_t row = z.first + i * z.step;
        const float m = z.ml[row].x;
        if (m == kNegInf) continue;  // no key in this part (its row may not even be written)
        const float f = ex2(m - all.x);
        float v[D / 32];
        load_row<D>(z.o + row * D, lane, v);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] += f * v[e];
      }
    };
    if (all.x != kNegInf) {
      add(x);
      add(y);
    }
    // A row without a key: 0.  (A NaN maximum or sum stays one.)
    const float inv = all.x == kNegInf ? 0.f : 1.f / all.y;
    const int t = r / p.G, h = hk * p.G + r % p.G;
    uint16_t* dst = static_cast<uint16_t*>(p.o) + b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2];
    if constexpr (D == 96) {
#pragma unroll
      for (int e = 0; e < 3; ++e) dst[3 * lane + e] = static_cast<uint16_t>(pack2<kBF16>(acc[e] * inv, 0.f));
    } else {
      uint32_t w[D / 64];
#pragma unroll
      for (int e = 0; e < D / 64; ++e) w[e] = pack2<kBF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      if constexpr (D == 64) *reinterpret_cast<uint32_t*>(dst + 2 * lane) = w[0];
      if constexpr (D == 128) *reinterpret_cast<uint2*>(dst + 4 * lane) = make_uint2(w[0], w[1]);
      if constexpr (D == 256) *reinterpret_cast<uint4*>(dst + 8 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }

  // Weights: sum over the rows of 2^(x - lse), lse = +inf for a row without a key.
  constexpr int kRows = 64;
  __shared__ float lse[kRows];
  const int j = key0 + 4 * threadIdx.x;
  float got[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < p.R; r0 += kRows) {
    const int rows = min(kRows, p.R - r0);
    __syncthreads();
    for (int r = wid; r < rows; r += kJoinThreads / 32) {
      const float2 all = total_of(prefix_parts(r0 + r), own_parts(r0 + r));
      if (lane == 0) lse[r] = all.x == kNegInf ? INFINITY : all.x + log2f(all.y);
    }
    __syncthreads();
    if (j < keys) {
      const float* row = p.logits + ((static_cast<int64_t>(b) * p.Hk + hk) * p.R + r0) * p.logits_ld + j;
      for (int r = 0; r < rows; ++r, row += p.logits_ld) {
        const float4 x = *reinterpret_cast<const float4*>(row);
        const float sub = lse[r];
        got[0] += ex2(x.x - sub);
        got[1] += ex2(x.y - sub);
        got[2] += ex2(x.z - sub);
        got[3] += ex2(x.w - sub);
      }
    }
  }
  if (j < keys) {
    float* w = p.weights + b * p.weights_stride[0] + hk * p.weights_stride[1] + j;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < keys) w[e] += got[e];
  }
}

// `overlap`: the grid may start before the kernel ahead of it in the stream is through.
template <typename K, typename... Args>
cudaError_t launch_with(K kernel, dim3 grid, int threads, size_t smem, bool overlap, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, bool kBF16, bool kMask>
cudaError_t launch_decode_t(const DecodeParams& p, int ctas, bool after_prefix, cudaStream_t s) {
  auto kern = decode_kernel<D, kBF16, kMask>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeShape<D>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_with(kern, dim3(ctas), 32 * kDecodeWarps, DecodeShape<D>::kBytes, after_prefix, s, p);
}

template <int D>
cudaError_t launch_decode_d(const DecodeParams& p, bool bf16, int ctas, bool after_prefix, cudaStream_t s) {
  if (p.mask) return bf16 ? launch_decode_t<D, true, true>(p, ctas, after_prefix, s)
                          : launch_decode_t<D, false, true>(p, ctas, after_prefix, s);
  return bf16 ? launch_decode_t<D, true, false>(p, ctas, after_prefix, s)
              : launch_decode_t<D, false, false>(p, ctas, after_prefix, s);
}

template <int D>
cudaError_t launch_join_d(const DecodeParams& p, bool bf16, cudaStream_t s) {
  const int rows = (p.R + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  const int adds = p.weights ? (p.C + kJoinKeys - 1) / kJoinKeys : 0;
  const dim3 grid(rows + adds, p.Hk, p.B);
  return bf16 ? launch_with(join_kernel<D, true>, grid, kJoinThreads, 0, true, s, p, rows)
              : launch_with(join_kernel<D, false>, grid, kJoinThreads, 0, true, s, p, rows);
}

}  // namespace

int decode_ctas_per_sm(int D) { return D == 256 ? DecodeShape<256>::kCtas : DecodeShape<128>::kCtas; }

cudaError_t launch_decode(const DecodeParams& p, int D, bool bf16, int ctas, bool after_prefix, cudaStream_t s) {
  if (D == 64) return launch_decode_d<64>(p, bf16, ctas, after_prefix, s);
  if (D == 96) return launch_decode_d<96>(p, bf16, ctas, after_prefix, s);
  if (D == 128) return launch_decode_d<128>(p, bf16, ctas, after_prefix, s);
  return launch_decode_d<256>(p, bf16, ctas, after_prefix, s);
}

cudaError_t launch_join(const DecodeParams& p, int D, bool bf16, cudaStream_t s) {
  if (D == 64) return launch_join_d<64>(p, bf16, s);
  if (D == 96) return launch_join_d<96>(p, bf16, s);
  if (D == 128) return launch_join_d<128>(p, bf16, s);
  return launch_join_d<256>(p, bf16, s);
}

}  // namespace fa4d
