// fa4d_prefix.cu — attention of a whole batch's new tokens over the prefix that its requests
// share: the rows of all requests and of the query heads of a KV head form one matrix, so the
// prefix is read once for all of them and both products run on the tensor cores.
//
// A CTA takes up to 256 rows of a KV head and a run of 128-key tiles, and writes its
// unnormalised output rows in 32 bits with their running maxima and sums; join_kernel joins
// the runs with the requests' own keys.  384 threads as in the forward kernel:
//   warp 0      K and V tiles by TMA into a ring each
//   warp 1      tcgen05.mma issuer
//   warp 2      tensor memory; at D = 256 the V producer
//   warps 4-7   slot 0: Q into shared memory, softmax, output (one thread per row)
//   warps 8-11  slot 1
// A slot is a chain S -> softmax -> P -> PV -> next S, about 3400 clocks a key tile alone and
// 3800 beside another slot, so two run per CTA.  With more than 128 rows they hold 128 rows
// each and share the K and V tiles; with at most 128 they hold the same rows and take even
// and odd key tiles (kSplitKeys), since then the bytes of K and V bound the kernel: one slot
// alone would take 64 KB per 3400 clocks, 5.5 TB/s over the GPU, two take 9.6 TB/s.  At
// D = 256 tensor memory holds one slot with two S buffers.
// Measured, with the decode and join kernels behind: 86 us for 512 rows a KV head x 32768 keys,
// Hk8 D128 (69 GFLOP, 0.8 PFLOP/s; a tile of 256 rows 2.05 us), 20 us for 128 rows x 4096 keys.  A
// tile's time is neither the chain's alone (halves of a tile with S buffers of their own, the next
// S always there ahead: no faster at D 64, 5% slower at D 128) nor the exponentials' (a third of
// them by polynomial: no change).  In short runs the start, Q and the output rows count (6 us a CTA).
// Tensor memory (512 columns): S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [256+D,256+2D); P
// (16-bit, rounded to the type of V as the product takes it) overwrites S.
#include "fa4d.h"
#include "fa4d_decode.h"
#include "fa4d_launch.cuh"
#include "fa4d_mma.cuh"
#include "fa4d_ptx.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 384;
// 384 x 168 registers at launch: 112 for the control warpgroup, 192 for the two softmax ones.
constexpr uint32_t kRegsCtl = 112, kRegsSoftmax = 192, kRegsLaunch = 168;
static_assert(128 * kRegsCtl + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "register split exceeds the launch");
constexpr float kNegInf = -INFINITY;
// O is rescaled only when a running maximum grows by more than this (log2 units).
constexpr float kRescaleThreshold = 8.0f;

// A whole 32-byte sector.
__device__ __forceinline__ void st_sector(float* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int D, bool kSplitKeys>
struct PrefixLayout {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kSlots = D == 256 ? 1 : 2;
  static constexpr int kQTiles = (D == 256 || kSplitKeys) ? 1 : 2;
  static constexpr int kStages = D == 256 ? 1 : D == 64 ? 4 : kSplitKeys ? 3 : 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kQTiles * kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kBar = kV + kStages * kTile;
  static constexpr int kNumBars = 8 + 4 * kStages;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kAlloc = kMisc + 16 + 1024;  // slack to align the base to 1024 B
  static_assert(kAlloc <= 232448, "shared memory beyond the 227 KB per-block limit");
};

template <int D, bool kBF16, bool kSplitKeys>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const __grid_constant__ PrefixParams p) {
  using L = PrefixLayout<D, kSplitKeys>;
  constexpr bool kDoubleS = L::kSlots == 1;
  constexpr int KVS = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* s_full = bars + 0;   // [2] per slot (per S buffer at D = 256)
  uint64_t* p_full = bars + 2;   // [2]
  uint64_t* o_full = bars + 4;   // [2]
  uint64_t* mma_drain = bars + 6;
  uint64_t* pv_done = bars + 7;  // D = 256: PV of a tile completed
  uint64_t* k_full = bars + 8;
  uint64_t* k_empty = k_full + KVS;
  uint64_t* v_full = k_empty + KVS;
  uint64_t* v_empty = v_full + KVS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  int* abort_flag = reinterpret_cast<int*>(smem + L::kMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y;
  const int row0 = blockIdx.x * 128 * L::kQTiles;
  const int tiles = (p.P + 127) / 128;
  int* runs_shared = reinterpret_cast<int*>(smem + L::kMisc + 8);
  // The start, side by side: the number of runs, barriers, tensor memory, Q.
  if (warp == 0) {
    pdl_wait();
    const int64_t units = line_before(p.lengths, p.C, p.B, lane, p.unit_shift) * p.Hk * p.load.row_tiles;
    const int r = choose_runs<D>(p.load, units, lane).runs;
    if (lane == 0) *runs_shared = r;
  } else if (warp == 1) {
    if (lane == 0) {
      prefetch_tmap(&p.tm_k);
      prefetch_tmap(&p.tm_v);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 128);
        mbar_init(&o_full[i], 1);
      }
      mbar_init(mma_drain, 1);
      mbar_init(pv_done, 1);
      for (int i = 0; i < KVS; ++i) {
        mbar_init(&k_full[i], 1);
        mbar_init(&k_empty[i], 1);
        mbar_init(&v_full[i], 1);
        mbar_init(&v_empty[i], 1);
      }
      *abort_flag = 0;
      fence_mbar_init();
    }
  } else if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (warp >= 4) {
    // Q rows into the swizzled tiles, D / 8 lanes a row, divided over the eight warps; lane i
    // knows where row i lies.  All copies are in flight at once and take no registers (loads,
    // eight a thread in flight: 1.2 to 2.9 us more a call at D 128 and 256).
    pdl_wait();
    constexpr int kRowsOfWarp = 16 * L::kQTiles, kLanes = D / 8, kRowsAtOnce = 32 / kLanes;
    const int first = (warp - 4) * kRowsOfWarp, row = row0 + first + (lane & (kRowsOfWarp - 1));
    const int token = row / p.G, h = hk * p.G + row % p.G;
    const int b = token / p.T, tt = token - b * p.T;
    const int64_t mine = b * p.q_stride[0] + tt * p.q_stride[1] + h * p.q_stride[2];
    const int c = lane % kLanes;
    uint8_t* dst = smem + L::kQ + (first >> 7) * L::kTile + (c >> 3) * 16384;
#pragma unroll 8
    for (int i = 0; i < kRowsOfWarp; i += kRowsAtOnce) {
      const int r = i + lane / kLanes;
      const int64_t at = __shfl_sync(0xffffffffu, mine, r);
      const bool some = row0 + first + r < p.rows && 8 * c < p.d_in;
      cp_async16(dst + ((first & 127) + r) * 128 + (((c ^ r) & 7) << 4), static_cast<const uint16_t*>(p.q) + (some ? at + 8 * c : 0),
                 some ? 16 : 0);
    }
    cp_async_wait_all();
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int runs = *runs_shared;
  if (static_cast<int>(blockIdx.z) >= runs) {
    if (warp == 2) tmem_dealloc(tmem, 512);
    return;
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.shares->parts = runs * (kSplitKeys ? 2 : 1);
  // Key tiles of this run, [kt0, kt0 + n): n >= 1.
  const int kt0 = static_cast<int>(static_cast<int64_t>(tiles) * blockIdx.z / runs);
  const int n = static_cast<int>(static_cast<int64_t>(tiles) * (blockIdx.z + 1) / runs) - kt0;
  // Whether slot 1 has rows (or tiles) of its own.
  const bool two = !kDoubleS && (kSplitKeys ? n > 1 : row0 + 128 < p.rows);
  pdl_launch();  // the decode kernel takes the SMs that are left, and these as their CTAs end

  if (warp < 4) {
    regs_dec<kRegsCtl>();
    auto produce = [&](const CUtensorMap* map, uint8_t* ring, uint64_t* full, uint64_t* empty, int u) {
      const int s = u % KVS;
      if (!mbar_wait(&empty[s], ((u / KVS) & 1) ^ 1, abort_flag)) return false;
      mbar_arrive_expect_tx(&full[s], L::kTile);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(ring + s * L::kTile + c * 16384, map, &full[s], c * 64, (kt0 + u) * 128, hk, 0);
      return true;
    };
    // Abort path: the copies of the last `upto` tiles must have landed before the CTA ends.
    auto settle = [&](uint64_t* full, int upto) {
      for (int j = max(0, upto - KVS); j < upto; ++j) mbar_wait_short(&full[j % KVS], (j / KVS) & 1);
    };
    if (warp == 0) {
      if (lane == 0) {
        int uk = 0, uv = 0;
        bool ok = true;
        for (int u = 0; ok && u < n; ++u) {
          ok = produce(&p.tm_k, smem + L::kK, k_full, k_empty, u);
          if (ok) uk = u + 1;
          if (!kDoubleS && ok) {
            ok = produce(&p.tm_v, smem + L::kV, v_full, v_empty, u);
            if (ok) uv = u + 1;
          }
        }
        if (*reinterpret_cast<volatile int*>(abort_flag)) {
          settle(k_full, uk);
          settle(v_full, uv);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      const uint32_t sQ = smem_u32(smem + L::kQ), sK = smem_u32(smem + L::kK), sV = smem_u32(smem + L::kV);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      };
      // S of tile u for slot t (S buffer t), and PV of tile u.
      auto qk = [&](int t, int u) {
        issue_qk<D, kBF16>(tmem + 128 * t, sQ + (L::kQTiles == 2 ? t * L::kTile : 0), sK + (u % KVS) * L::kTile);
        tc_commit(&s_full[t]);
      };
      auto pv = [&](int t, int u, bool accumulate) {
        issue_pv<D, kBF16>(kDoubleS ? tmem + 256 : tmem + 256 + D * t, tmem + 128 * t, sV + (u % KVS) * L::kTile, accumulate);
      };
      bool ok = wait(&k_full[0], 0);
      if (ok) {
        tc_fence_after();
        if (elect_one()) {
          qk(0, 0);
          if (!kSplitKeys && two) qk(1, 0);
          tc_commit(&k_empty[0]);
        }
        __syncwarp();
      }
      if constexpr (kDoubleS || kSplitKeys) {
        // One chain, or two on alternate tiles.  D = 256: tile u's S in buffer u & 1, S of
        // tile u + 1 issued ahead of PV of tile u.  kSplitKeys: tile u belongs to slot u & 1,
        // whose next S (tile u + 2) follows its PV.
        constexpr int kAheadTiles = kDoubleS ? 1 : 2;
        if (kSplitKeys && ok && n > 1) {
          ok = wait(&k_full[1 % KVS], (1 / KVS) & 1);
          if (ok) {
            tc_fence_after();
            if (elect_one()) {
              qk(1, 1);
              tc_commit(&k_empty[1 % KVS]);
            }
            __syncwarp();
          }
        }
        for (int u = 0; ok && u < n; ++u) {
          const int un = u + kAheadTiles, t = u & 1;
          auto next_s = [&]() {
            if (un >= n) return true;
            if (!wait(&k_full[un % KVS], (un / KVS) & 1)) return false;
            tc_fence_after();
            if (elect_one()) {
              qk(un & 1, un);
              tc_commit(&k_empty[un % KVS]);
            }
            __syncwarp();
            return true;
          };
          if (kDoubleS && !(ok = next_s())) break;
          ok = wait(&v_full[u % KVS], (u / KVS) & 1) && wait(&p_full[t], (u >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            pv(t, u, kDoubleS ? u > 0 : u > 1);
            if (kDoubleS) tc_commit(pv_done);
            tc_commit(&v_empty[u % KVS]);
            if (un >= n && (kSplitKeys || u + 1 == n)) tc_commit(&o_full[kDoubleS ? 0 : t]);
          }
          __syncwarp();
          if (kSplitKeys && !(ok = next_s())) break;
        }
      } else {
        for (int u = 0; ok && u < n; ++u) {
          const bool more = u + 1 < n;
          ok = wait(&v_full[u % KVS], (u / KVS) & 1);
          if (!ok) break;
          for (int t = 0; t < (two ? 2 : 1); ++t) {
            ok = wait(&p_full[t], u & 1);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              pv(t, u, u > 0);
              if (!more) tc_commit(&o_full[t]);
            }
            __syncwarp();
            if (more) {
              ok = t > 0 || wait(&k_full[(u + 1) % KVS], ((u + 1) / KVS) & 1);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) qk(t, u + 1);
              __syncwarp();
            }
          }
          if (!ok) break;
          if (elect_one()) {
            tc_commit(&v_empty[u % KVS]);
            if (more) tc_commit(&k_empty[(u + 1) % KVS]);
          }
          __syncwarp();
        }
      }
      // Every product must have completed before tensor memory is released.
      if (elect_one()) tc_commit(mma_drain);
      __syncwarp();
      wait(mma_drain, 0);
    } else if (kDoubleS && warp == 2) {
      if (lane == 0) {
        int uv = 0;
        for (; uv < n; ++uv)
          if (!produce(&p.tm_v, smem + L::kV, v_full, v_empty, uv)) break;
        if (*reinterpret_cast<volatile int*>(abort_flag)) settle(v_full, uv);
      }
      __syncwarp();
    }
  } else {
    regs_inc<kRegsSoftmax>();
    const int t = (warp - 4) >> 2;
    const int quad = (warp & 3) * 32;
    const int row = row0 + (L::kQTiles == 2 ? 128 * t : 0) + quad + lane;
    const bool valid = row < p.rows;
    const bool warp_valid = row - lane < p.rows;  // some lane has a row
    const uint32_t lane_base = static_cast<uint32_t>(quad) << 16;
    // Columns of the output row, [c0, c0 + kCols): at D = 256 both warpgroups write the slot's.
    constexpr int kCols = kDoubleS ? D / 2 : D;
    auto write_row = [&](uint32_t tO, int64_t out, int c0) {
      if (!__all_sync(0xffffffffu, mbar_wait(&o_full[kDoubleS ? 0 : t], 0, abort_flag))) return;
      tc_fence_after();
      if (!warp_valid) return;
#pragma unroll
      for (int c = 0; c < kCols; c += 32) {
        uint32_t o[32];
        tmem_ld32(tO + c0 + c, o);
        tmem_wait_ld();
        if (valid && c0 + c < p.d_in) {
          float* dst = p.o + out * p.d_in + c0 + c;
#pragma unroll
          for (int v = 0; v < 4; ++v) st_sector(dst + 8 * v, &o[8 * v]);
        }
      }
    };
    if (t < L::kSlots && (t == 0 || two || kSplitKeys)) {
      const int count = kSplitKeys ? (n - t + 1) / 2 : n;
      const uint32_t tO = tmem + lane_base + 256 + (kDoubleS ? 0 : D * t);
      float m_run = kNegInf, l_run = 0.f;
      bool ok = true;
      int i = 0;
      for (; i < count; ++i) {
        const int kbase = (kt0 + (kSplitKeys ? 2 * i + t : i)) * 128;
        const int sb = kDoubleS ? (i & 1) : t;
        const uint32_t tS = tmem + lane_base + 128 * sb;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[sb], kDoubleS ? (i >> 1) & 1 : i & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (warp_valid) {
          auto online_update = [&](float m_tile) {
            const float m_new = fmaxf(m_run, m_tile);
            const bool need = m_new > m_run + kRescaleThreshold;
            float alpha = 1.f;
            if (need) {
              alpha = ex2(m_run - m_new);  // m_run == -inf -> 0
              l_run *= alpha;
              m_run = m_new;
            }
            if (i > 0 && __any_sync(0xffffffffu, need)) {
              // The slot's previous PV has completed (this S was issued after it); with two S
              // buffers it is waited for.
              if (kDoubleS) mbar_wait(pv_done, (i - 1) & 1, abort_flag);
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(tO + 16 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                tmem_st16(tO + 16 * c, o);
              }
            }
            return m_run == kNegInf ? 0.f : m_run;
          };
          uint32_t x[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[32 * c]));
          tmem_wait_ld();
          float m4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
          // A full tile takes the maximum of the raw logits and folds the scale into the
          // exponent's FMA; the last tile of the prefix, and a scale that is not positive,
          // scale first.
          float sc, m_use;
          if (kbase + 128 <= p.P && p.scale_log2 > 0.f) {
#pragma unroll
            for (int k = 0; k < 128; k += 2)
              m4[(k >> 1) & 3] = fmax3(m4[(k >> 1) & 3], __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
            sc = p.scale_log2;
            m_use = online_update(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc);
          } else {
#pragma unroll
            for (int k = 0; k < 128; ++k) {
              const float v = kbase + k < p.P ? __uint_as_float(x[k]) * p.scale_log2 : kNegInf;
              x[k] = __float_as_uint(v);
              m4[k & 3] = fmaxf(m4[k & 3], v);
            }
            sc = 1.f;
            m_use = online_update(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
          }
          const uint64_t sc2 = f2(sc, sc), nm2 = f2(-m_use, -m_use);
          uint64_t rs2 = f2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 a =
                  f2_split(ffma2(f2(__uint_as_float(x[32 * c + 2 * k]), __uint_as_float(x[32 * c + 2 * k + 1])), sc2, nm2));
              const float p0 = ex2(a.x), p1 = ex2(a.y);
              rs2 = fadd2(rs2, f2(p0, p1));
              pk[k] = pack2<kBF16>(p0, p1);
            }
            tmem_st16(tS + 16 * c, pk);
          }
          const float2 rs = f2_split(rs2);
          l_run += rs.x + rs.y;
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&p_full[sb]);
      }

      // This run's part of the row; one without a tile is marked by its maximum, -inf, and sum, 0.
      if (count > 0) part_of_keys(m_run, l_run);
      const int part = kSplitKeys ? 2 * blockIdx.z + t : blockIdx.z;
      const int64_t out = (static_cast<int64_t>(hk) * p.parts + part) * p.rows + row;
      if (valid) p.ml[out] = make_float2(m_run, l_run);
      if (count > 0 && ok) write_row(tO, out, 0);
      tc_fence_before();
    } else if (kDoubleS) {
      const int64_t out = (static_cast<int64_t>(hk) * p.parts + blockIdx.z) * p.rows + row;
      write_row(tmem + lane_base + 256, out, kCols);
      tc_fence_before();
    }
  }

  __syncthreads();
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int*>(abort_flag)) atomicOr(p.status, FA4D_DEV_TIMEOUT_PREFIX);
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool kBF16, bool kSplitKeys>
cudaError_t launch_prefix_t(const PrefixParams& p, int Hk, int splits, cudaStream_t s) {
  using L = PrefixLayout<D, kSplitKeys>;
  auto kern = prefix_kernel<D, kBF16, kSplitKeys>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
  if (e != cudaSuccess) return e;
  const dim3 grid((p.rows + 128 * L::kQTiles - 1) / (128 * L::kQTiles), Hk, splits);
  return launch_chained(kern, grid, kThreads, L::kAlloc, 1, s, p);
}

template <int D, bool kBF16>
cudaError_t launch_prefix_d(const PrefixParams& p, int Hk, int splits, bool split_keys, cudaStream_t s) {
  if constexpr (D != 256)
    if (split_keys) return launch_prefix_t<D, kBF16, true>(p, Hk, splits, s);
  return launch_prefix_t<D, kBF16, false>(p, Hk, splits, s);
}

}  // namespace

cudaError_t launch_prefix(const PrefixParams& p, int D, bool bf16, int Hk, int splits, bool split_keys, cudaStream_t s) {
  if (D == 64) return bf16 ? launch_prefix_d<64, true>(p, Hk, splits, split_keys, s)
                           : launch_prefix_d<64, false>(p, Hk, splits, split_keys, s);
  if (D == 256) return bf16 ? launch_prefix_d<256, true>(p, Hk, splits, split_keys, s)
                            : launch_prefix_d<256, false>(p, Hk, splits, split_keys, s);
  return bf16 ? launch_prefix_d<128, true>(p, Hk, splits, split_keys, s)
              : launch_prefix_d<128, false>(p, Hk, splits, split_keys, s);
}

}  // namespace fa4d
