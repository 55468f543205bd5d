// fa4d_decode.cu — attention of a few new tokens over long caches: the keys are divided over
// all warps of the GPU (decode_kernel), and the partial results joined (join_kernel).
//
// o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m), x_j = scale log2(e) q.k_j: numerator and
// denominator over any set of keys, each with its own m, are joined exactly by factors
// 2^(m - m_all).
#include "fa4d.h"
#include "fa4d_decode.h"
#include "fa4d_launch.cuh"
#include "fa4d_line.cuh"

namespace fa4d {

namespace {

constexpr float kNegInf = -INFINITY;

template <int D>
struct DecodeShape {
  static constexpr int kBoxes = (D + 63) / 64;       // TMA boxes of 64 columns (96: zeros past it)
  static constexpr int kBox = kUnitKeys * 128;       // 128-byte rows, 16-byte chunks swizzled
  static constexpr int kTile = kBoxes * kBox;        // K or V of a unit
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = D == 64 ? 6 : 3;
  // At head dim 256 the queries stay in shared memory: in registers (64, beside 128 of output)
  // they spilled, and no product's operands were loaded ahead of it (524 MB of own keys, B32
  // Hq16 Hk16: 204 us so, 182 from shared memory; 16 requests of 6 tokens: 5.8 us less a call).
  static constexpr bool kQShared = D == 256;
  static constexpr int kQ = kDecodeWarps * kStages * kStage;
  static constexpr int kBars = kQ + (kQShared ? kDecodeWarps * kTile : 0);
  static constexpr int kBytes = kBars + kDecodeWarps * kStages * 8 + 8 + 1024;  // aligned to 1024
  static_assert(kBytes <= 232448, "shared memory beyond the 227 KB per-block limit");
  // 16-byte chunk c of row `row` of a tile.
  static __device__ __forceinline__ uint32_t at(int row, int c) {
    return (c >> 3) * kBox + row * 128 + (((c ^ row) & 7) << 4);
  }
};

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
// One warp: its units in order, each 16 keys of K and V brought by TMA into the warp's own ring
// (no barrier between warps), x = Q K^T and P V by m16n8k16 products with the fp32 output row
// tile in registers.  Memory bounds it, at 16 FLOP per byte of K and V for a row tile of 16: 1208
// MB of own keys (B128 Hk8 D128, 512 to 4096 entries) in 200-205 us with the join, 5.9-6.0 TB/s,
// 92% of the measured copy rate.  Short calls are bound by the start: lengths, division, first
// loads take about 4 us, a unit 0.6 to 1.0 us (head dim 64 to 256) when memory is idle.  A row
// tile is the product's 16 rows: more tiles of a request read its keys again, from L2.
template <int D, bool kBF16, bool kMask>
__global__ void __launch_bounds__(32 * kDecodeWarps, kDecodeCtas<D>) decode_kernel(
    const __grid_constant__ DecodeParams p, bool after_prefix) {
  using S = DecodeShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * kDecodeWarps + wid;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars) + wid * S::kStages;
  int* abort_flag = reinterpret_cast<int*>(smem + S::kBars + kDecodeWarps * S::kStages * 8);
  if (lane < S::kStages) mbar_init(&full[lane], 1);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    prefetch_tmap(&p.tm_k);
    prefetch_tmap(&p.tm_v);
  }
  fence_mbar_init();
  __syncthreads();
  // Behind the prefix kernel, every CTA of which has seen everything ahead complete, and which
  // writes nothing that is read here, there is nothing to wait for.
  if (!after_prefix) pdl_wait();
  pdl_launch();

  Lengths<kUnitShift> lengths;
  lengths.load(p, lane);
  const int64_t total = static_cast<int64_t>(p.prefix_tiles) * p.Hk * (p.prefix_units + kPrefixItemUnits) +
                        lengths.line(p, lane) * p.Hk * p.tiles;
  const Shares shares = shares_of<D>(p, total, lane);
  if (warp == 0 && lane == 0) {
    p.shares->early = shares.early;
    p.shares->each = shares.each;
    p.shares->late = shares.late;
  }
  const int64_t first = warp_start(shares, warp);
  const int64_t run = min(warp_start(shares, warp + 1), total) - first;
  Place<kUnitShift> at;
  at.left = 0;
  if (run > 0) at = find_place(p, lengths, first, run, lane);
  if (at.more()) {
    uint8_t* ring = smem + wid * S::kStages * S::kStage;
    uint8_t* queries = smem + S::kQ + wid * S::kTile;  // kQShared
    Place<kUnitShift> in = at;

    // K and V of the unit at `in` into a stage.  Rows past the item's keys come along (zeros past
    // the cache's end).
    auto bring = [&](int stage) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[stage], S::kStage);
        uint8_t* dst = ring + stage * S::kStage;
        const CUtensorMap* k = in.prefix ? &p.tm_pk : &p.tm_k;
        const CUtensorMap* v = in.prefix ? &p.tm_pv : &p.tm_v;
        const int b = in.prefix ? 0 : in.b;
#pragma unroll
        for (int c = 0; c < S::kBoxes; ++c) {
          tma_load_4d(dst + c * S::kBox, k, &full[stage], c * 64, in.u * kUnitKeys, in.hk, b);
          tma_load_4d(dst + S::kTile + c * S::kBox, v, &full[stage], c * 64, in.u * kUnitKeys, in.hk, b);
        }
      }
    };

    int brought = 0;
    auto bring_next = [&]() {
      if (in.more()) {
        bring(brought % S::kStages);
        ++brought;
        in.advance(p, lengths);
      }
    };

    uint32_t qf[S::kQShared ? 1 : D / 16][4];
    float acc[D / 8][4];
    float m[2], l[2];
    unsigned seen;           // bit i: row i has seen one of this thread's keys
    int lim[2];              // keys below lim[i] are seen by row i of this thread
    const uint8_t* mrow[2];  // its mask row
    float* lrow[2];          // its row of logits, null where there is none
    const int col = 2 * (lane & 3);

    auto begin_item = [&]() {
      seen = 0;
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
        const uint16_t* row = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
        if constexpr (S::kQShared) {  // a row's four lanes take every fourth chunk
          if (!valid) row = static_cast<const uint16_t*>(p.q);
#pragma unroll
          for (int c = lane & 3; c < D / 8; c += 4)
            cp_async16(queries + S::at((lane >> 2) + 8 * i, c), row + 8 * c, valid ? 16 : 0);
        } else {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][i] = valid ? __ldcg(reinterpret_cast<const uint32_t*>(row + col + 16 * kk)) : 0u;
            qf[kk][i + 2] = valid ? __ldcg(reinterpret_cast<const uint32_t*>(row + col + 16 * kk + 8)) : 0u;
          }
        }
        m[i] = kNegInf;
        l[i] = 0.f;
      }
      if constexpr (S::kQShared) {
        cp_async_wait_all();
        __syncwarp();
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
        // A maximum of -inf over keys that were seen (part_of_keys, fa4d_decode.h).
        const unsigned saw = __ballot_sync(0xffffffffu, (seen >> i) & 1u);
        if ((saw >> (lane & 28)) & 15u) part_of_keys(m[i], l[i]);
        const int r = (lane >> 2) + 8 * i;
        if (r >= p.seg_rows) continue;
        const int64_t row = seg * p.seg_rows + r;
        if ((lane & 3) == 0) p.seg_ml[row] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<float2*>(p.seg_o + row * D + 8 * c + col) = make_float2(acc[c][2 * i], acc[c][2 * i + 1]);
      }
    };

    // Mask bits of a unit for this thread's two rows: bit 4 i + 2 nt + e for row i, key
    // 8 nt + col + e.  They are loaded a unit ahead.
    auto mask_bits = [&](int u) {
      uint32_t bits = 0xffu;
      if constexpr (kMask) {
        if (at.prefix) return bits;
        uint8_t v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int j = min(u * kUnitKeys + 8 * ((x >> 1) & 1) + col + (x & 1), at.keys - 1);
          v[x] = mrow[x >> 2] ? __ldcg(mrow[x >> 2] + j) : 0;
        }
        bits = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) bits |= (v[x] != 0 ? 1u : 0u) << x;
      }
      return bits;
    };

    uint32_t keep_next = 0;
    // The first rounds only bring (one copy of that code: a CTA runs for microseconds, and
    // instructions fetched for the first time are a good part of its start).
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) bring_next();
    begin_item();
    keep_next = mask_bits(at.u);
#pragma unroll 1
    for (int it = 0; at.more(); ++it) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[it % S::kStages], (it / S::kStages) & 1, abort_flag))) {
        // Given up: what is still on its way must land before the CTA ends.
        for (int j = it; j < brought; ++j) mbar_wait_short(&full[j % S::kStages], (j / S::kStages) & 1);
        break;
      }
      bring_next();  // into the stage of the unit before this one
      const uint32_t keep_bits = keep_next;
      if (kMask && at.u + 1 < at.units) keep_next = mask_bits(at.u + 1);
      const uint32_t sk = smem_u32(ring) + (it % S::kStages) * S::kStage, sv = sk + S::kTile;

      float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(sk + S::at(row, 2 * kk + half), kf);
          uint32_t(&q)[4] = qf[S::kQShared ? 0 : kk];
          if constexpr (S::kQShared) ldsm4(smem_u32(queries) + S::at(lane & 15, 2 * kk + (lane >> 4)), q);
          mma16816<kBF16>(x[0], q, kf[0], kf[1]);
          mma16816<kBF16>(x[1], q, kf[2], kf[3]);
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
          const bool keep = j < lim[i] && (!kMask || ((keep_bits >> (4 * i + 2 * nt + (e & 1))) & 1u));
          x[nt][e] = keep ? x[nt][e] * p.scale_log2 : kNegInf;
          if (keep) {
            dead &= ~(1u << kj);
            seen |= 1u << i;
          }
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
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + S::at(row, c)),
                         "r"(0)
                         : "memory");
        }
        fence_async_smem();  // before a copy into the stage
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
          ldsm4_t(sv + S::at(row, 2 * c + half), vf);
          mma16816<kBF16>(acc[2 * c], pf, vf[0], vf[1]);
          mma16816<kBF16>(acc[2 * c + 1], pf, vf[2], vf[3]);
        }
      }
      if (at.u + 1 == at.units || at.left == 1) end_item();
      if (at.advance(p, lengths) && at.more()) {
        begin_item();
        keep_next = mask_bits(at.u);
      }
    }
  }
  if (lane == 0 && *reinterpret_cast<volatile int*>(abort_flag)) atomicOr(p.status, FA4D_DEV_TIMEOUT_PREFIX);
  // The join may start once this grid is through, and must then also find what the prefix
  // kernel before it wrote: one CTA stays until that is done (all of them staying would keep
  // the SMs from the CTAs still to come).
  if (after_prefix && blockIdx.x + 1 == gridDim.x) pdl_wait();
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

constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
// Partial rows of a warp in flight (16 at head dim 64: Hq64 Hk1 B48 35.3 -> 33.9 us; at 256 the
// registers cost more: draft trees of B16 35.4 -> 36.7).
template <int D>
constexpr int kJoinAhead = D == 64 ? 16 : 8;
constexpr int kWeighRows = 4;                 // rows of weights taken together
constexpr int kWeighKeys = 4 * kJoinThreads;  // own keys of a block of weigh_kernel at a time
constexpr int kWeighTimes = 4;
// Rows whose sums weigh_kernel works out itself, beside the join (16 requests, Hk4, prefix 2050, own
// up to 770: 24 rows at D 256 33.0 us so, 34.5 behind it; 64 rows at D 128 49.1 and 42.7).
constexpr int kWeighOwnRows = 32;

// The partial results of the rows of (request b, KV head hk).
struct Joined {
  const DecodeParams& p;
  int b, hk, keys;
  int64_t each, first;
  Shares shares;

  // Before the partial results are there: what the lengths tell.  `divide`: the division too, as
  // decode_kernel works it out where no prefix kernel runs beside it.
  __device__ __forceinline__ Joined(const DecodeParams& params, int b_, int hk_, int lane, bool divide) : p(params), b(b_), hk(hk_) {
    keys = length_of(p, b);
    each = static_cast<int64_t>(p.groups) * p.tiles;
    const int64_t prefix_all = static_cast<int64_t>(p.prefix_tiles) * p.groups * (p.prefix_units + kPrefixItemUnits);
    first = prefix_all + line_before(p.lengths, p.C, b, lane, p.unit_shift) * each;
    if (divide)
      shares = even_shares(prefix_all + line_before(p.lengths, p.C, p.B, lane, p.unit_shift) * each, p.warps, p.min_units);
  }
  // Of an item of `count` units that starts at `from` on the line.
  __device__ __forceinline__ Parts of_units(int64_t from, int count, int64_t item, int row) const {
    Parts x{p.seg_o, p.seg_ml, 0, static_cast<int64_t>(p.heads) * p.seg_rows, 0};
    if (count > 0) {
      const int64_t w0 = warp_of(shares, from);
      x.n = static_cast<int>(warp_of(shares, from + count - 1) - w0 + 1);
      x.first = (((w0 + item) << p.head_shift) + (hk & (p.heads - 1))) * p.seg_rows + row;
    }
    return x;
  }
  __device__ __forceinline__ void load_shares() {
    const int4 s = __ldcg(reinterpret_cast<const int4*>(p.shares));
    shares = Shares{s.x, s.y, s.z, s.w};
  }
  // The parts of row r: of its own keys, and of the prefix.
  __device__ __forceinline__ Parts own(int r) const {
    const int64_t i = static_cast<int64_t>(hk >> p.head_shift) * p.tiles + r / 16;
    return of_units(first + i * line_of(keys, p.unit_shift), units_of(keys, p.unit_shift), static_cast<int64_t>(p.prefix_tiles) * p.groups + b * each + i, r % 16);
  }
  __device__ __forceinline__ Parts prefix(int r) const {
    const int64_t row = static_cast<int64_t>(b) * p.R + r;
    if (p.splits)
      return Parts{p.pre_o, p.pre_ml, static_cast<int64_t>(hk) * p.splits * p.pre_rows + row, p.pre_rows, shares.parts};
    const int64_t i = static_cast<int64_t>(hk) * p.prefix_tiles + row / 16;
    return of_units(i * (p.prefix_units + kPrefixItemUnits), p.prefix_tiles ? p.prefix_units : 0, i, static_cast<int>(row % 16));
  }
};

// log2 of a row's sum from its maximum and sum; +inf for a row without a key.
__device__ __forceinline__ float log2_sum(float m, float l) {
  return m == kNegInf ? (l == 0.f ? INFINITY : NAN) : m + log2f(l);
}

// Joins the output: row_warps warps a row, each a share of its parts.  Everything here is
// latency: partial rows are loaded ahead of the maximum that scales them (about 3 us for 42 parts
// of 32 rows, 8 us behind a decode kernel of 296 CTAs at B32 Hq32).
template <int D, bool kBF16, bool kDivide>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ DecodeParams p, int row_warps) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  Joined at(p, blockIdx.z, blockIdx.y, lane, kDivide);
  const int r = (blockIdx.x * (blockDim.x / 32) + wid) / row_warps;
  Parts x{}, y{};
  if constexpr (!kDivide) {
    pdl_wait();
    pdl_launch();
    at.load_shares();
  }
  if (r < p.R) {
    x = at.prefix(r);
    y = at.own(r);
  }
  if constexpr (kDivide) {
    pdl_wait();
    pdl_launch();
  }
  const int share = (x.n + y.n + row_warps - 1) / row_warps;
  const int n0 = min(wid % row_warps * share, x.n + y.n), n = min(n0 + share, x.n + y.n);
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  float m_all = kNegInf, l_all = 0.f;
  bool undefined = false;  // a part of keys of logit -inf
  // 32 parts at a time, lane i with the maximum of part i; their rows kJoinAhead at a time.
  for (int i0 = n0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    float2 ml = make_float2(kNegInf, 0.f);
    if (i < n) ml = i < x.n ? x.ml[x.first + i * x.step] : y.ml[y.first + (i - x.n) * y.step];
    float f;
    auto settle = [&]() {  // this batch's maximum, factors and sum; the output so far rescaled
      float mx = ml.x;
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mx = fmaxf(mx, m_all);
      f = ml.x == kNegInf ? 0.f : ex2(ml.x - mx);
      undefined = undefined || (ml.x == kNegInf && ml.y != 0.f);
      float l = ml.y * f;
#pragma unroll
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const float old = m_all == kNegInf ? 0.f : ex2(m_all - mx);
      l_all = l_all * old + l;
      m_all = mx;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] *= old;
    };
    const int batch = min(32, n - i0);
    for (int j0 = 0; j0 < batch; j0 += kJoinAhead<D>) {
      float v[kJoinAhead<D>][D / 32];
#pragma unroll
      for (int u = 0; u < kJoinAhead<D>; ++u) {
        const int j = min(i0 + j0 + u, n - 1);
        const float* row = j < x.n ? x.o + (x.first + j * x.step) * D : y.o + (y.first + (j - x.n) * y.step) * D;
        load_row<D>(row, lane, v[u]);
      }
      if (j0 == 0) settle();
#pragma unroll
      for (int u = 0; u < kJoinAhead<D>; ++u) {
        // A part without a key (maximum -inf) may not even have its row written.
        const float fu = __shfl_sync(0xffffffffu, f, j0 + u), mu = __shfl_sync(0xffffffffu, ml.x, j0 + u);
        if (j0 + u < batch && mu != kNegInf) {
#pragma unroll
          for (int e = 0; e < D / 32; ++e) acc[e] += fu * v[u][e];
        }
      }
    }
  }
  if (__any_sync(0xffffffffu, undefined) && m_all == kNegInf) l_all = 1.f;
  if (row_warps > 1) {  // the row's first warp adds the others'
    __shared__ float others[kJoinWarps][D];
    __shared__ float2 others_ml[kJoinWarps];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) others[wid][(D / 32) * lane + e] = acc[e];
    if (lane == 0) others_ml[wid] = make_float2(m_all, l_all);
    __syncthreads();
    if (wid % row_warps) return;
    float mx = kNegInf;
    for (int i = 0; i < row_warps; ++i) mx = fmaxf(mx, others_ml[wid + i].x);
    l_all = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    for (int i = 0; i < row_warps; ++i) {
      const float2 ml = others_ml[wid + i];
      if (ml.x == kNegInf) {
        if (mx == kNegInf) l_all = fmaxf(l_all, ml.y);
        continue;
      }
      const float fi = ex2(ml.x - mx);
      l_all += fi * ml.y;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += fi * others[wid + i][(D / 32) * lane + e];
    }
    m_all = mx;
  }
  if (r >= p.R) return;
  // A row without a key: 0.  One whose every logit is -inf, or that saw a NaN (in l_all): NaN.
  const float inv = m_all == kNegInf ? (l_all == 0.f ? 0.f : NAN) : 1.f / l_all;
  if (p.weights && lane == 0) p.lse[(static_cast<int64_t>(at.b) * p.Hk + at.hk) * p.R + r] = log2_sum(m_all, l_all);
  const int t = r / p.G, h = at.hk * p.G + r % p.G;
  uint16_t* dst = static_cast<uint16_t*>(p.o) + at.b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2];
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
}

// What a key of logit x gains: nothing where the row does not see it (-inf), even if the row's sum
// is NaN.
__device__ __forceinline__ float gain(float x, float lse) { return x == kNegInf ? 0.f : ex2(x - lse); }

// Adds to the weights of a request's own keys: the sum over the rows of 2^(x - lse), lse = +inf
// for a row without a key.  A kernel of its own beside join_kernel, whose registers would leave
// it two blocks an SM (33 us in one kernel at B128 Hk8, 4096 slots; 95 MB).  It starts when
// every block of join_kernel has found the partial results complete, so they are complete here,
// works beside it, and its last block waits so that this kernel is over only when that one is.
// With more than kWeighOwnRows rows, a warp's turns at their sums take longer than waiting for
// join_kernel, which has them all.  Four blocks an SM: 64 registers a thread, no spills (16 requests
// of 6 tokens, D 256, own 6-770: 39.1 us a call with five, 36.8 with four).
__global__ void __launch_bounds__(kJoinThreads, 4) weigh_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kRows = 64;
  __shared__ float lse[kRows];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  Joined at(p, blockIdx.z, blockIdx.y, lane, false);
  const int key0 = blockIdx.x * kWeighTimes * kWeighKeys + 4 * threadIdx.x;
  float* weights = p.weights + at.b * p.weights_stride[0] + at.hk * p.weights_stride[1];
  if (blockIdx.x * kWeighTimes * kWeighKeys < at.keys) {
    const bool from_join = p.R > kWeighOwnRows;
    if (from_join)
      pdl_wait();
    else
      at.load_shares();
    float* first_row = p.logits + (static_cast<int64_t>(at.b) * p.Hk + at.hk) * p.R * p.logits_ld;
    for (int r0 = 0; r0 < p.R; r0 += kRows) {
      const int rows = min(kRows, p.R - r0);
      const float* logits = first_row + static_cast<int64_t>(r0) * p.logits_ld;
      float4 x[kWeighRows];
      auto load = [&](int j, int r) {
#pragma unroll
        for (int u = 0; u < kWeighRows; ++u)
          x[u] = __ldcg(reinterpret_cast<const float4*>(logits + static_cast<int64_t>(min(r + u, rows - 1)) * p.logits_ld + j));
      };
      __syncthreads();
      if (from_join && threadIdx.x < rows)
        lse[threadIdx.x] = p.lse[(static_cast<int64_t>(at.b) * p.Hk + at.hk) * p.R + r0 + threadIdx.x];
      for (int r = wid; !from_join && r < rows; r += kJoinWarps) {
        // Maximum and sum over all parts of the row.
        const Parts px = at.prefix(r0 + r), py = at.own(r0 + r);
        float m = kNegInf, l = 0.f;
        for (int i = lane; i < px.n + py.n; i += 32) {
          const float2 ml = __ldcg(i < px.n ? px.ml + px.first + i * px.step : py.ml + py.first + (i - px.n) * py.step);
          const float mx = fmaxf(m, ml.x);
          l = mx != kNegInf ? l * ex2(m - mx) + ml.y * ex2(ml.x - mx) : fmaxf(l, ml.y);
          m = mx;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
          const float mx = fmaxf(m, m2);
          l = mx != kNegInf ? l * ex2(m - mx) + l2 * ex2(m2 - mx) : fmaxf(l, l2);
          m = mx;
        }
        if (lane == 0) lse[r] = log2_sum(m, l);
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < kWeighTimes; ++i) {
        const int j = key0 + i * kWeighKeys;
        if (j >= at.keys) break;
        // The gain, complete before it meets the weight: added to a large weight row by row, gains
        // below its last place would be lost (64 rows of 3e-6 beside 100: all of them).  The weight
        // is on its way meanwhile (loaded after the rows: 1.3 us more a call).  Between batches of
        // rows the gain waits in the first row's place, whose logits have been read.
        float4* sums = reinterpret_cast<float4*>(first_row + j);
        float got[4] = {0.f, 0.f, 0.f, 0.f}, had[4];
        const bool whole = p.weights_vec && j + 4 <= at.keys;
        if (whole) {
          const float4 w = __ldcg(reinterpret_cast<const float4*>(weights + j));
          had[0] = w.x, had[1] = w.y, had[2] = w.z, had[3] = w.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) had[e] = j + e < at.keys ? __ldcg(weights + j + e) : 0.f;
        }
        if (r0) {
          const float4 s = *sums;
          got[0] = s.x, got[1] = s.y, got[2] = s.z, got[3] = s.w;
        }
        for (int r = 0; r < rows; r += kWeighRows) {
          load(j, r);
#pragma unroll
          for (int u = 0; u < kWeighRows; ++u) {
            const float sub = r + u < rows ? lse[r + u] : INFINITY;
            got[0] += gain(x[u].x, sub);
            got[1] += gain(x[u].y, sub);
            got[2] += gain(x[u].z, sub);
            got[3] += gain(x[u].w, sub);
          }
        }
        if (r0 + rows < p.R) {
          *sums = make_float4(got[0], got[1], got[2], got[3]);
        } else if (whole) {
          *reinterpret_cast<float4*>(weights + j) =
              make_float4(had[0] + got[0], had[1] + got[1], had[2] + got[2], had[3] + got[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + e < at.keys) weights[j + e] = had[e] + got[e];
        }
      }
    }
  }
  pdl_launch();
  if (blockIdx.x + 1 == gridDim.x && blockIdx.y + 1 == gridDim.y && blockIdx.z + 1 == gridDim.z) pdl_wait();
}

template <int D, bool kBF16, bool kMask>
cudaError_t launch_decode_t(const DecodeParams& p, int ctas, bool after_prefix, cudaStream_t s) {
  auto kern = decode_kernel<D, kBF16, kMask>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeShape<D>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, dim3(ctas), 32 * kDecodeWarps, DecodeShape<D>::kBytes, 1, s, p, after_prefix);
}

template <int D>
cudaError_t launch_decode_d(const DecodeParams& p, bool bf16, int ctas, bool after_prefix, cudaStream_t s) {
  if (p.mask) return bf16 ? launch_decode_t<D, true, true>(p, ctas, after_prefix, s)
                          : launch_decode_t<D, false, true>(p, ctas, after_prefix, s);
  return bf16 ? launch_decode_t<D, true, false>(p, ctas, after_prefix, s)
              : launch_decode_t<D, false, false>(p, ctas, after_prefix, s);
}

template <int D>
cudaError_t launch_join_d(const DecodeParams& p, bool bf16, int sms, cudaStream_t s) {
  // Warps a row: as many as leave the grid about one block an SM (B32 Hq32 took 4 us longer
  // with four of them and four times the blocks; one request 2 us less with eight).
  int row_warps = 1;
  while (row_warps < kJoinWarps && 2LL * row_warps * p.R * p.Hk * p.B <= 8LL * sms) row_warps *= 2;
  const int all = p.R * row_warps, blocks = (all + kJoinWarps - 1) / kJoinWarps;
  // Blocks without idle warps where there are more than the SMs hold at once (three each), since
  // those keep registers from others (512 blocks of 4 rows: 31.1 -> 28.0 us, 1024: 98.6 -> 96).
  // Otherwise whole blocks: smaller ones crowd on the SMs that the decode kernel leaves first
  // (256 blocks of 4 rows: 47.3 us so, 48.2 with 4 warps).
  int warps = kJoinWarps;
  if (static_cast<int64_t>(blocks) * p.Hk * p.B > 3LL * sms)
    warps = ((all + blocks - 1) / blocks + row_warps - 1) / row_warps * row_warps;
  const dim3 grid(blocks, p.Hk, p.B);
  // Few blocks work the division out while decode_kernel's last CTAs run, which spares them a wait
  // (1 request, 4000 own keys in 8 bits: 10.8 us a call so for 9.8, 16 requests of 24 rows 39.2 and
  // 38.3); of many the division holds up what is still running (48 requests of 64 rows, 384 blocks:
  // 33.6 us and 37.0).
  const bool divide = !p.load.items && static_cast<int64_t>(blocks) * p.Hk * p.B <= 2LL * sms;
  auto kern = divide ? (bf16 ? join_kernel<D, true, true> : join_kernel<D, false, true>)
                     : (bf16 ? join_kernel<D, true, false> : join_kernel<D, false, false>);
  const cudaError_t e = launch_chained(kern, grid, 32 * warps, 0, 1, s, p, row_warps);
  if (e != cudaSuccess || !p.weights) return e;
  const dim3 weigh((p.C + kWeighTimes * kWeighKeys - 1) / (kWeighTimes * kWeighKeys), p.Hk, p.B);
  return launch_chained(weigh_kernel, weigh, kJoinThreads, 0, 1, s, p);
}

}  // namespace

cudaError_t launch_decode(const DecodeParams& p, int D, bool bf16, int ctas, bool after_prefix, cudaStream_t s) {
  if (D == 64) return launch_decode_d<64>(p, bf16, ctas, after_prefix, s);
  if (D == 96) return launch_decode_d<96>(p, bf16, ctas, after_prefix, s);
  if (D == 128) return launch_decode_d<128>(p, bf16, ctas, after_prefix, s);
  return launch_decode_d<256>(p, bf16, ctas, after_prefix, s);
}

cudaError_t launch_join(const DecodeParams& p, int D, bool bf16, int sms, cudaStream_t s) {
  if (D == 64) return launch_join_d<64>(p, bf16, sms, s);
  if (D == 96) return launch_join_d<96>(p, bf16, sms, s);
  if (D == 128) return launch_join_d<128>(p, bf16, sms, s);
  return launch_join_d<256>(p, bf16, sms, s);
}

}  // namespace fa4d
