// fa4d_decode8.cu — attention of a few new tokens over long caches held in 8 bits: decode8_kernel
// makes the partial results that join_kernel (fa4d_decode.cu) joins.
//
// With codes k, v and the scales s, z of their blocks: x_j = (scale log2(e) s_j) q.k_j and
// o = sum_j 2^(x_j - m) z_j v_j / sum_j 2^(x_j - m).  Codes go to the products as fp16, which holds
// them exactly; a scale, one for the 64 slots of a block, multiplies logits, and weights before their
// rounding.  What is rounded are the weights 2^(x_j + log2 z_j - n), under a running maximum n of
// their own: so a block of large scale that gets no weight takes no bits from the others.
//
// Weights are rounded to fp16, 11 bits, because the product with V takes them so: a second product of what the
// rounding leaves would double that one's work.  Errors against 64 bits, with weights so and in 32 bits (root of
// the mean square, of that of the outputs): bf16 outputs 1.63e-3 and 1.62e-3, fp16 outputs 2.3e-4 and
// 2.1e-4.  Sums of the probabilities and all partial rows are in 32 bits.
#include <cuda_fp16.h>

#include "fa4d.h"
#include "fa4d_cache8.cuh"
#include "fa4d_decode.h"
#include "fa4d_launch.cuh"
#include "fa4d_line.cuh"
#include "fa4d_ptx.cuh"

namespace fa4d {

namespace {

constexpr float kNegInf = -INFINITY;
// Probabilities are computed 2^kRaise times as large, so that their factors to weights (up to 2^126, where
// V's scales are far apart) reach all that 32 bits hold.
constexpr int kRaise = 16;

template <int D, int kCols>
struct Shape8 {
  static constexpr int kShift = kUnit8Shift<D>;
  static constexpr int kKeys = 1 << kShift;          // of a unit: 8 KB of K and V
  static constexpr int kWide = D == 96 ? 128 : D;    // columns computed (96: zeros past it)
  static constexpr int kRow = D == 64 ? 64 : 128;    // bytes of a row of a TMA box
  static constexpr int kBoxes = kWide / kRow;
  static constexpr int kBox = kKeys * kRow;
  static constexpr int kTile = kBoxes * kBox;        // K or V of a unit
  static constexpr int kStage = 2 * kTile;
  // Where the output takes 128 registers the queries stay in shared memory: in registers (64) they
  // spilled.
  static constexpr bool kQShared = kWide * kCols == 512;
  static constexpr int kStages = (kQShared || kCtas8<D, kCols> == 3 ? 16384 : 24576) / kStage;
  static constexpr int kQ = kDecodeWarps * kStages * kStage;  // [warp][column tile][step][lane] 8 bytes
  static constexpr int kBars = kQ + (kQShared ? kDecodeWarps * kCols * kWide * 16 : 0);
  static constexpr int kBytes = kBars + kDecodeWarps * kStages * 8 + 8 + 1024;  // aligned to 1024
  static constexpr int kKeyTiles = kKeys / 16;       // 16-key tiles of a unit
  static constexpr int kSteps = kWide / 64;          // 64 columns: four steps of the product with Q
  static constexpr int kOutTiles = kWide / 16;       // 16-column tiles of the output
  // 16-byte chunk c of row `row` of a tile: 128-byte rows are swizzled, 64-byte rows are not.
  static __device__ __forceinline__ uint32_t at(int row, int c) {
    return D == 64 ? row * 64 + c * 16 : (c >> 3) * kBox + row * 128 + (((c ^ row) & 7) << 4);
  }
};

// Rows of a product's 16-key tile hold its keys in this order (of 8), so that lanes which load
// together find their chunks in different banks; what is done with the keys does not depend on it.
__device__ __forceinline__ int key_of(int i) { return (i & 1) * 4 + (i >> 1); }

// Plain loads and unordered products: the compiler interleaves them.
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds8(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
// An 8 x 8 matrix of 16-bit elements transposed, two elements of a row a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c (16 x 8, fp32) += a (16 x 16) b (16 x 8), fp16
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One warp: its units in order, each 8 KB of K and V brought by TMA into the warp's own ring, keys
// along the 16 rows of a product and kCols * 8 query rows along its columns: S^T = K Q^T and
// O^T = V^T P^T.  A lane reads 16 codes of a key at once, converts them in registers to the
// product's operands (of V, two keys' bytes are interleaved first, which transposes it), and P^T
// turns between the products by movmatrix.
//
// With up to 8 rows memory bounds it: 1.21 GB of e4m3 codes (B64 Hk8 D128, 2048 to 16384 entries, 4
// rows) 186 us with the join, 6.5 TB/s, 99% of the measured copy rate, in both layouts; int8 188.  With
// 16 rows a unit's conversions, softmax and waits do (about 1000 instructions and 1.7 us of two warps a
// scheduler, D 64): 48 requests of 64 rows, 26 MB read four times, 33.6 us, of which the join 7 and the
// start 4; tiles of 32 rows, which read the keys half as often, took 41, for fewer warps share the
// work.  Units of head dim 256 (16 keys) take 1.9 us: 16 requests of 24 rows, own up to 2050, 38 us.
template <int D, bool kInt8, int kCols, bool kMask>
__global__ void __launch_bounds__(32 * kDecodeWarps, kCtas8<D, kCols>) decode8_kernel(
    const __grid_constant__ Decode8Params p8, bool after_prefix) {
  using S = Shape8<D, kCols>;
  constexpr int kShift = S::kShift;
  const DecodeParams& p = p8.d;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kDecodeWarps / p.heads) + wid / p.heads;
  const int sub = wid % p.heads;  // of the heads that its neighbours take along
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
  // Behind the prefix kernel there is nothing to wait for (as in decode_kernel).
  if (!after_prefix) pdl_wait();
  pdl_launch();

  Lengths<kShift> lengths;
  lengths.load(p, lane);
  const int64_t total = lengths.line(p, lane) * p.groups * p.tiles;
  const Shares shares = shares_of<D>(p, total, lane);
  if (warp == 0 && sub == 0 && lane == 0) {
    p.shares->early = shares.early;
    p.shares->each = shares.each;
    p.shares->late = shares.late;
  }
  const int64_t first = warp_start(shares, warp);
  const int64_t run = min(warp_start(shares, warp + 1), total) - first;
  Place<kShift> at;
  at.left = 0;
  if (run > 0) at = find_place(p, lengths, first, run, lane);
  if (at.more()) {
    uint8_t* ring = smem + wid * S::kStages * S::kStage;
    Place<kShift> in = at;

    int brought = 0;
    auto bring_next = [&]() {
      if (!in.more()) return;
      if (lane == 0) {
        uint64_t* bar = &full[brought % S::kStages];
        mbar_arrive_expect_tx(bar, S::kStage);
        uint8_t* dst = ring + brought % S::kStages * S::kStage;
#pragma unroll
        for (int c = 0; c < S::kBoxes; ++c) {
          tma_load_4d(dst + c * S::kBox, &p.tm_k, bar, c * S::kRow, in.u << kShift, in.hk * p.heads + sub, in.b);
          tma_load_4d(dst + S::kTile + c * S::kBox, &p.tm_v, bar, c * S::kRow, in.u << kShift, in.hk * p.heads + sub, in.b);
        }
      }
      ++brought;
      in.advance(p, lengths);
    };

    uint32_t qf[kCols][S::kQShared ? 1 : S::kSteps][8];
    uint8_t* queries = smem + S::kQ + wid * kCols * S::kWide * 16 + lane * 8;  // kQShared
    float acc[S::kOutTiles][kCols][4];
    // Of columns 2 q4 and 2 q4 + 1 of each tile of 8 query rows:
    float qs[kCols][2];      // scale log2(e), and what the row was divided by for fp16
    float m[kCols][2];       // running maximum of the logits
    float n[kCols][2];       // of the weights that go to the product with V
    float l[kCols][2];       // this lane's part of the sum, 2^kRaise times as large
    int lim[kCols][2];       // keys below it are seen
    const uint8_t* mrow[kCols][2];
    unsigned seen;           // bit 2 c + e: the column has seen one of this lane's keys
    int whole;               // units that end at or below this key are seen by all rows
    const float* ks;         // scales of the item's blocks
    const float* vs;

    auto begin_item = [&]() {
      const int hk = at.hk * p.heads + sub;
      seen = 0;
      whole = kMask ? 0 : p.causal ? at.keys - p.T + 1 : at.keys;
      ks = p8.k_scale + at.b * p8.k_scale_stride[0] + hk * p8.k_scale_stride[1];
      vs = p8.v_scale + at.b * p8.v_scale_stride[0] + hk * p8.v_scale_stride[1];
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int r = at.tile * 16 + 8 * c + g;
        const bool valid = r < p.R;
        const int t = r / p.G, h = hk * p.G + r % p.G;
        const uint16_t* row = static_cast<const uint16_t*>(p.q) + at.b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
        // Each lane 16 elements of every 64, the columns of the codes that it reads.
        uint4 raw[S::kSteps][2];
#pragma unroll
        for (int j = 0; j < S::kSteps; ++j) {
          const int col = 64 * j + 16 * q4;
          const bool ok = valid && col < D;
          raw[j][0] = ok ? __ldcg(reinterpret_cast<const uint4*>(row + col)) : make_uint4(0, 0, 0, 0);
          raw[j][1] = ok ? __ldcg(reinterpret_cast<const uint4*>(row + col) + 1) : make_uint4(0, 0, 0, 0);
        }
        // In fp16 under the power of two that brings the row's largest magnitude to 2^15..2^16: what
        // falls below fp16's steps then is below 2^-39 of that one.
        uint32_t most = 0;
        auto value = [&](uint32_t w) { return p8.q_bf16 ? unpack2<true>(w) : unpack2<false>(w); };
#pragma unroll
        for (int j = 0; j < S::kSteps; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = value(reinterpret_cast<const uint32_t*>(raw[j])[i]);
            most = max(most, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
          }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = static_cast<int>(most >> 23);  // biased; 255 where an element is not finite
        // 2^(142 - e): by two factors where one would pass fp32's range.
        const int up = e == 0 ? 0 : 142 - e;
        const float f0 = __uint_as_float(static_cast<uint32_t>(127 + up / 2) << 23);
        const float f1 = e == 255 ? NAN : __uint_as_float(static_cast<uint32_t>(127 + up - up / 2) << 23);
#pragma unroll
        for (int j = 0; j < S::kSteps; ++j)
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float2 v = value(reinterpret_cast<const uint32_t*>(raw[j])[i]);
            const float2 u = value(reinterpret_cast<const uint32_t*>(raw[j])[i + 1]);
            const uint2 h = make_uint2(pack2<false>(v.x * f0 * f1, v.y * f0 * f1), pack2<false>(u.x * f0 * f1, u.y * f0 * f1));
            if constexpr (S::kQShared)
              *reinterpret_cast<uint2*>(queries + ((c * S::kSteps + j) * 4 + i / 2) * 256) = h;  // read by this lane alone
            else
              qf[c][j][i] = h.x, qf[c][j][i + 1] = h.y;
          }
        const float back = 1.f / f0 / f1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          qs[c][x] = p.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * q4 + 4 * x);
          const int rx = at.tile * 16 + 8 * c + 2 * q4 + x;
          const int tx = rx / p.G, hx = hk * p.G + rx % p.G;
          lim[c][x] = rx >= p.R ? 0 : p.causal ? at.keys - p.T + tx + 1 : at.keys;
          if (kMask)
            mrow[c][x] = rx >= p.R ? nullptr
                                   : p.mask + at.b * p.mask_stride[0] + hx * p.mask_stride[1] + tx * p.mask_stride[2];
          m[c][x] = n[c][x] = kNegInf;
          l[c][x] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < S::kOutTiles; ++i)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][c][e] = 0.f;
    };

    auto end_item = [&]() {
      const int64_t seg = (warp + at.item(p)) * p.heads + sub;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) seen |= __shfl_xor_sync(0xffffffffu, seen, o);
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l[c][x] += __shfl_xor_sync(0xffffffffu, l[c][x], o);
          // The output row under the maximum of the logits; a part without weights is 0.
          const float to = n[c][x] == kNegInf ? 1.f : ex2(n[c][x] - m[c][x]);
          l[c][x] *= 1.f / (1 << kRaise);
          if ((seen >> (2 * c + x)) & 1u) part_of_keys(m[c][x], l[c][x]);
          const int r = 8 * c + 2 * q4 + x;
          if (r >= p.seg_rows) continue;
          const int64_t row = seg * p.seg_rows + r;
          if (g == 0) p.seg_ml[row] = make_float2(m[c][x], l[c][x]);
          float* o = p.seg_o + row * D;
          // 16 columns a lane of each 128 (8 of 64): elements 2 i and 2 i + 1 from tile i.
          constexpr int kPer = D == 64 ? 4 : 8;
#pragma unroll
          for (int h = 0; h < S::kOutTiles / kPer; ++h) {
            const int col = D == 64 ? 8 * g : 128 * h + 16 * key_of(g);
            if (col >= D) continue;
#pragma unroll
            for (int i = 0; i < kPer; i += 2) {
              const float(&a)[4] = acc[h * kPer + i][c];
              const float(&b)[4] = acc[h * kPer + i + 1][c];
              *reinterpret_cast<float4*>(o + col + 2 * i) = make_float4(a[x] * to, a[2 + x] * to, b[x] * to, b[2 + x] * to);
            }
          }
        }
    };

    // The mask's bytes of this lane's logits of a unit, loaded a unit ahead and looked at then.
    constexpr int kMaskBytes = kMask ? S::kKeyTiles * kCols * 4 : 1;
    uint8_t mask_now[kMaskBytes], mask_next[kMaskBytes];
    auto load_mask = [&](int u) {
      if constexpr (kMask) {
#pragma unroll
        for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = min((u << kShift) + 16 * i + 8 * (e >> 1) + key_of(g), at.keys - 1);
              mask_next[(i * kCols + c) * 4 + e] = mrow[c][e & 1] ? __ldcg(mrow[c][e & 1] + j) : 0;
            }
      }
    };
    auto keep_now = [&](int i, int c, int e) { return mask_now[kMask ? (i * kCols + c) * 4 + e : 0] != 0; };
    // Scales of a unit, loaded a unit ahead too.
    auto scales = [&](int u) {
      const int i = (u << kShift) / FA4D_CACHE_BLOCK;
      return make_float2(__ldcg(ks + i), __ldcg(vs + i));
    };

    float2 scale_next;
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) bring_next();
    bool fresh = true;  // at an item's first unit (one copy of that code, too)
#pragma unroll 1
    for (int it = 0; at.more(); ++it) {
      if (fresh) {
        begin_item();
        load_mask(at.u);
        scale_next = scales(at.u);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&full[it % S::kStages], (it / S::kStages) & 1, abort_flag))) {
        // Given up: what is still on its way must land before the CTA ends.
        for (int j = it; j < brought; ++j) mbar_wait_short(&full[j % S::kStages], (j / S::kStages) & 1);
        break;
      }
      bring_next();  // into the stage of the unit before this one
#pragma unroll
      for (int i = 0; i < kMaskBytes; ++i) mask_now[i] = mask_next[i];
      const float2 scale = scale_next;
      if (at.u + 1 < at.units) {
        load_mask(at.u + 1);
        scale_next = scales(at.u + 1);
      }
      const uint8_t* sk = ring + (it % S::kStages) * S::kStage;
      const uint8_t* sv = sk + S::kTile;

      // Few tiles would be few chains of dependent products: those have two sums.
      constexpr int kChains = S::kKeyTiles * kCols <= 2 ? 2 : 1;
      float x[S::kKeyTiles][kCols][4], x2[kChains == 2 ? S::kKeyTiles : 1][kCols][4];
#pragma unroll
      for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[i][c][e] = 0.f;
            if (kChains == 2) x2[kChains == 2 ? i : 0][c][e] = 0.f;
          }
#pragma unroll
      for (int j = 0; j < S::kSteps; ++j) {
#pragma unroll
        for (int i = 0; i < S::kKeyTiles; ++i) {
          const uint4 lo = lds16(sk + S::at(16 * i + key_of(g), 4 * j + q4));
          const uint4 hi = lds16(sk + S::at(16 * i + 8 + key_of(g), 4 * j + q4));
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t a0, a1, a2, a3;
            codes_to_half2<kInt8>(wl[k], a0, a2);
            codes_to_half2<kInt8>(wh[k], a1, a3);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              uint2 q;
              if constexpr (S::kQShared)
                q = lds8(queries + ((c * S::kSteps + j) * 4 + k) * 256);
              else
                q = make_uint2(qf[c][j][2 * k], qf[c][j][2 * k + 1]);
              mma16(kChains == 2 && (k & 1) ? x2[kChains == 2 ? i : 0][c] : x[i][c], a0, a1, a2, a3, q.x, q.y);
            }
          }
        }
      }
      if (kChains == 2)
#pragma unroll
        for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][c][e] += x2[kChains == 2 ? i : 0][c][e];

      // -inf where the row does not see the key.
      const int key0 = at.u << kShift;
      const bool all_seen = key0 + S::kKeys <= whole;
      if (all_seen) {
        seen = 0xffffffffu;
      } else {
        uint64_t live = 0;  // keys that a row sees
#pragma unroll
        for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int kj = 16 * i + 8 * (e >> 1) + key_of(g);
              const bool keep = key0 + kj < lim[c][e & 1] && (!kMask || keep_now(i, c, e));
              if (keep) {
                live |= 1ull << kj;
                seen |= 1u << (2 * c + (e & 1));
              } else {
                x[i][c][e] = kNegInf;
              }
            }
        // A key that no row sees may hold anything: its V is cleared, since 0 * NaN is NaN (int8
        // has none).
        if constexpr (!kInt8) {
          const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(live));
          const uint32_t hi = S::kKeys > 32 ? __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(live >> 32)) : 0u;
          constexpr uint32_t kAll = S::kKeys < 32 ? (1u << (S::kKeys & 31)) - 1u : 0xffffffffu;
          if (lo != kAll || (S::kKeys > 32 && hi != kAll)) {
            constexpr int kChunks = S::kWide / 16;
#pragma unroll 1
            for (int id = lane; id < S::kKeys * kChunks; id += 32) {
              const int row = id / kChunks, ch = id - row * kChunks;
              if (!(((row < 32 ? lo : hi) >> (row & 31)) & 1u))
                *reinterpret_cast<uint4*>(const_cast<uint8_t*>(sv) + S::at(row, ch)) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();  // before a copy into the stage
            __syncwarp();
          }
        }
      }

      // Running maxima; sums and outputs are rescaled only where one grew.
      float zl = __log2f(scale.y);
      float f[kCols][2];  // to log2 units
      bool odd = zl != zl;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[c][e] = qs[c][e] * scale.x;
          odd = odd || !(f[c][e] > 0.f);
        }
      if (odd) {
        // A factor below 0 goes to the logits, and one of 0, which -inf would make NaN; NaN, of it or of
        // the scale of the values, reaches the sums of the rows that see one of the keys.
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& u = f[c][e];
#pragma unroll
            for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
              for (int h = 0; h < 4; h += 2) {
                float& y = x[i][c][e + h];
                if (y == kNegInf) continue;
                if (u != u || zl != zl) l[c][e] = NAN;
                y = u != u ? kNegInf : u < 0.f ? -y : u == 0.f ? 0.f : y;
              }
            u = u < 0.f ? -u : u > 0.f ? u : 1.f;
          }
        if (zl != zl) zl = kNegInf;
      }
      // A maximum follows the logits only when they pass it by more than 2^kSlack (so weights stay far
      // below fp16's largest), which one vote over the lanes' own maxima tells: then they are brought
      // together, and sums and output rescaled.
      constexpr float kSlack = 8.f;
      static_assert(kRaise > kSlack, "the factors of weights whose probability is above 2^-126 stay below 2^126");
      float mx[kCols][2];
      bool past = false;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x_max = kNegInf;
#pragma unroll
          for (int i = 0; i < S::kKeyTiles; ++i) x_max = fmaxf(x_max, fmaxf(x[i][c][e], x[i][c][e + 2]));
          mx[c][e] = x_max * f[c][e];
          past = past || mx[c][e] > m[c][e] + kSlack || mx[c][e] + zl > n[c][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, past)) {
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          float to[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y = mx[c][e];
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            const float m_new = fmaxf(m[c][e], y), n_new = fmaxf(n[c][e], y + zl);
            l[c][e] *= m[c][e] == m_new ? 1.f : ex2(m[c][e] - m_new);
            to[e] = n[c][e] == n_new ? 1.f : ex2(n[c][e] - n_new);
            m[c][e] = m_new;
            n[c][e] = n_new;
          }
#pragma unroll
          for (int i = 0; i < S::kOutTiles; ++i) {
            acc[i][c][0] *= to[0];
            acc[i][c][1] *= to[1];
            acc[i][c][2] *= to[0];
            acc[i][c][3] *= to[1];
          }
        }
      }
      float w_of[kCols][2], under[kCols][2];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          under[c][e] = (m[c][e] == kNegInf ? 0.f : m[c][e]) - kRaise;
          // From a probability under m to a weight under n.  A weight is at most 2^kSlack (see above), so a
          // probability whose factor is cut off here is below 2^(kSlack - 126 - kRaise) = 2^-134: 0 in 32 bits.
          // The maxima's difference first, which is exact or nearly: added to V's scale, large logits would lose
          // the last bits of either.
          w_of[c][e] = ex2(fminf(under[c][e] - (n[c][e] == kNegInf ? 0.f : n[c][e]) + zl, 126.f));
        }
      uint32_t pf[S::kKeyTiles][kCols][2];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < S::kKeyTiles; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = ex2(fmaf(x[i][c][2 * h], f[c][0], -under[c][0]));
            const float p1 = ex2(fmaf(x[i][c][2 * h + 1], f[c][1], -under[c][1]));
            l[c][0] += p0;
            l[c][1] += p1;
            pf[i][c][h] = transpose8(pack2<false>(p0 * w_of[c][0], p1 * w_of[c][1]));
          }

#pragma unroll
      for (int i = 0; i < S::kKeyTiles; ++i) {
        if constexpr (D == 64) {
          uint2 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = lds8(sv + (16 * i + q4 + 4 * k) * 64 + 8 * g);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t v0 = w ? v[0].y : v[0].x, v1 = w ? v[1].y : v[1].x, v2 = w ? v[2].y : v[2].x, v3 = w ? v[3].y : v[3].x;
            uint32_t a[2][4];
            codes_to_half2<kInt8>(__byte_perm(v0, v1, 0x5140), a[0][0], a[0][1]);
            codes_to_half2<kInt8>(__byte_perm(v2, v3, 0x5140), a[0][2], a[0][3]);
            codes_to_half2<kInt8>(__byte_perm(v0, v1, 0x7362), a[1][0], a[1][1]);
            codes_to_half2<kInt8>(__byte_perm(v2, v3, 0x7362), a[1][2], a[1][3]);
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
              for (int c = 0; c < kCols; ++c) mma16(acc[2 * w + o][c], a[o][0], a[o][1], a[o][2], a[o][3], pf[i][c][0], pf[i][c][1]);
          }
        } else {
#pragma unroll
          for (int half = 0; half < S::kBoxes; ++half) {
            uint32_t v[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 u = lds16(sv + S::at(16 * i + q4 + 4 * k, 8 * half + key_of(g)));
              v[k][0] = u.x, v[k][1] = u.y, v[k][2] = u.z, v[k][3] = u.w;
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t a[2][4];
              codes_to_half2<kInt8>(__byte_perm(v[0][w], v[1][w], 0x5140), a[0][0], a[0][1]);
              codes_to_half2<kInt8>(__byte_perm(v[2][w], v[3][w], 0x5140), a[0][2], a[0][3]);
              codes_to_half2<kInt8>(__byte_perm(v[0][w], v[1][w], 0x7362), a[1][0], a[1][1]);
              codes_to_half2<kInt8>(__byte_perm(v[2][w], v[3][w], 0x7362), a[1][2], a[1][3]);
#pragma unroll
              for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int c = 0; c < kCols; ++c)
                  mma16(acc[8 * half + 2 * w + o][c], a[o][0], a[o][1], a[o][2], a[o][3], pf[i][c][0], pf[i][c][1]);
            }
          }
        }
      }
      if (at.u + 1 == at.units || at.left == 1) end_item();
      fresh = at.advance(p, lengths);
    }
  }
  if (lane == 0 && *reinterpret_cast<volatile int*>(abort_flag)) atomicOr(p.status, FA4D_DEV_TIMEOUT_PREFIX);
  // One CTA stays until the prefix kernel is through (as in decode_kernel).
  if (after_prefix && blockIdx.x + 1 == gridDim.x) pdl_wait();
}

template <int D, bool kInt8, int kCols, bool kMask>
cudaError_t launch_t(const Decode8Params& p, int ctas, bool after_prefix, cudaStream_t s) {
  auto kern = decode8_kernel<D, kInt8, kCols, kMask>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape8<D, kCols>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, dim3(ctas), 32 * kDecodeWarps, Shape8<D, kCols>::kBytes, 1, s, p, after_prefix);
}

template <int D, bool kInt8>
cudaError_t launch_d(const Decode8Params& p, int ctas, bool after_prefix, cudaStream_t s) {
  if (decode8_cols(p.d.R) == 1)
    return p.d.mask ? launch_t<D, kInt8, 1, true>(p, ctas, after_prefix, s) : launch_t<D, kInt8, 1, false>(p, ctas, after_prefix, s);
  return p.d.mask ? launch_t<D, kInt8, 2, true>(p, ctas, after_prefix, s) : launch_t<D, kInt8, 2, false>(p, ctas, after_prefix, s);
}

}  // namespace

cudaError_t launch_decode8(const Decode8Params& p, int D, bool int8, int ctas, bool after_prefix, cudaStream_t s) {
  if (D == 64) return int8 ? launch_d<64, true>(p, ctas, after_prefix, s) : launch_d<64, false>(p, ctas, after_prefix, s);
  if (D == 96) return int8 ? launch_d<96, true>(p, ctas, after_prefix, s) : launch_d<96, false>(p, ctas, after_prefix, s);
  if (D == 128) return int8 ? launch_d<128, true>(p, ctas, after_prefix, s) : launch_d<128, false>(p, ctas, after_prefix, s);
  return int8 ? launch_d<256, true>(p, ctas, after_prefix, s) : launch_d<256, false>(p, ctas, after_prefix, s);
}

}  // namespace fa4d
