// fa4d_evict.cu — eviction from a cache by the attention weight its entries received: per
// (request, KV head) the entries to keep are found by radix selection on the weights, and K,
// V and weights copied together, in one launch.
//
// A cluster of CTAs takes one (request, KV head): each CTA histograms a slice of the weights,
// the histograms are added through distributed shared memory, and each CTA copies a slice of
// the kept entries.  Bound by memory: the kept rows of K and V are read and written once
// (4 D bytes each way), against 4 bytes of weight an entry.
#include "fa4d.h"
#include "fa4d_kernels.h"
#include "fa4d_launch.cuh"
#include "fa4d_ptx.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 8192;  // weights of a CTA at a time
constexpr int kBins = 2048;   // of a radix pass: 11, 11 and 10 bits of the weight
// Pieces of a row of K and of V that a thread has in flight (B32 Hk8 D128, 2304 slots to 1536:
// 78 us with 2, 74 with 3, 75 with 4, 80 with 6; less shared memory, for a larger L1: no change).
constexpr int kRowsInFlight = 3;
constexpr int kAhead = 4;  // other reads of a thread in flight

// Larger weight, larger key; -0 as 0; NaN below everything.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void add_cluster(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

struct Smem {
  alignas(16) uint32_t hist[kBins];
  alignas(16) uint32_t counts[4];  // of this CTA's slice: kept for sure, equal to the threshold
  uint32_t warp_sum[kWarps];
  uint32_t found[2];
  alignas(16) uint32_t total[2][kBins];  // rank 0's, of slices: the cluster's histogram of even and odd passes
  uint2 ballot[kChunk / 32];  // of each 32 entries: kept for sure, equal to the threshold
  uint32_t key[kChunk];   // order_key of the weights
  uint16_t list[kChunk];  // slots of this CTA's share (selection without slices)
};

// Sum of x over the threads before this one; `all` is the sum over the CTA.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* warp_sum, uint32_t& all) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  uint32_t upto = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t left = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += left;
  }
  __syncthreads();  // the sums of an earlier scan have been read
  if (lane == 31) warp_sum[wid] = upto;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const uint32_t s = warp_sum[i];
    if (i < wid) before += s;
    all += s;
  }
  return before + upto - x;
}

template <int VEC>
struct Piece;
template <>
struct Piece<8> {
  using T = uint4;
  static __device__ __forceinline__ T zero() { return make_uint4(0u, 0u, 0u, 0u); }
};
template <>
struct Piece<1> {
  using T = uint16_t;
  static __device__ __forceinline__ T zero() { return 0; }
};

// Caches of up to kChunk entries are selected by every CTA of the cluster for itself (the
// weights are a few hundredths of the rows, and nothing waits between CTAs); of longer ones
// each CTA takes a slice of the weights.  Their order keys stay in shared memory across the
// passes (re-read where a slice is longer than kChunk).  The loops are left rolled: with the
// keys in registers and every loop over them unrolled, each instruction ran once per CTA and
// its fetch was the time (2700 to 3300 clocks a radix pass and 8000 to 18000 for the slots at
// 1024 to 2304 entries; 2000 and 2400 now).  What is left is the copy: 63000 of 78000 clocks
// of a CTA at B32 Hk8 D128, 2304 slots to 1536 (74 us in all, 5.2 TB/s, 81% of the measured
// copy rate), 155000 of 195000 at B4 Hk8 D64, 65536 to 32768 (119 us, 4.7 TB/s, 72%).
template <int VEC>
__global__ void __launch_bounds__(kThreads, 2) evict_kernel(const __grid_constant__ fa4d_evict_args a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int rank = static_cast<int>(cluster_rank()), ranks = static_cast<int>(cluster_size());
  const int item = static_cast<int>(blockIdx.x) / ranks;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int b = item / a.Hk, h = item - b * a.Hk;
  pdl_wait();
  pdl_launch();
  const int n = min(max(__ldcg(a.lengths + b), 0), a.C);
  const int kept = min(n, a.keep);
  const float* w = a.weights + b * a.weights_stride[0] + h * a.weights_stride[1];
  float* w_out = a.weights_out + b * a.weights_out_stride[0] + h * a.weights_out_stride[1];
  int32_t* index = a.index_out + static_cast<int64_t>(item) * a.keep;
  if (h == 0 && rank == 0 && threadIdx.x == 0) a.lengths_out[b] = kept;

  const bool sliced = n > kChunk;
  const int share = (a.keep + ranks - 1) / ranks;
  const int slot0 = min(rank * share, a.keep), slot1 = min(slot0 + share, a.keep);

  if (n > a.keep) {
    // The middle [a.sinks, late) gives its `want` heaviest entries.
    const int late = n - a.recent;
    uint32_t want = a.keep - a.sinks - a.recent, threshold = 0;
    const bool none = want == 0;
    const int per = sliced ? (n + ranks - 1) / ranks : n;
    const int lo = sliced ? min(rank * per, n) : 0, hi = min(lo + per, n);
    const bool once = hi - lo <= kChunk;

    auto sync = [&]() {  // of everyone who works on this selection
      if (sliced)
        cluster_sync();
      else
        __syncthreads();
    };
    auto load = [&](int base) {
      const int end = min(hi, base + kChunk);
      for (int j0 = base + threadIdx.x; j0 < end; j0 += kAhead * kThreads) {
        float x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) x[u] = j0 + u * kThreads < end ? __ldcg(w + j0 + u * kThreads) : 0.f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (j0 + u * kThreads < end) sm.key[j0 + u * kThreads - base] = order_key(x[u]);
      }
    };
    load(lo);

    // Radix selection of the want-th largest key of the middle, from the top bits down.  With
    // slices, the CTAs add the bins that are not empty to rank 0's, which finds the digit for
    // all (each CTA adding all bins of all others cost 5 us a pass).
    if (!none) {
      constexpr int kMine = 4;  // bins of a thread in scans
      static_assert(kMine * kThreads == kBins, "");
      auto clear = [&](uint32_t* hist) {
        *reinterpret_cast<uint4*>(&hist[kMine * threadIdx.x]) = make_uint4(0u, 0u, 0u, 0u);
      };
      if (sliced) {
        clear(sm.total[0]);
        cluster_sync();
      }
#pragma unroll 1
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        clear(sm.hist);
        __syncthreads();
        for (int base = lo; base < hi; base += kChunk) {
          if (!once) load(base);  // every thread reads only what it wrote
          const int end = min(min(hi, late), base + kChunk);
          for (int j0 = base + threadIdx.x; j0 < end; j0 += kAhead * kThreads) {
            uint32_t key[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) key[u] = sm.key[min(j0 + u * kThreads, end - 1) - base];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
              const int j = j0 + u * kThreads;
              // Bits above this digit equal to the threshold's (pass 0 has none).
              if (j < end && j >= a.sinks && (pass == 0 || (key[u] >> (shift + bits)) == threshold))
                atomicAdd(&sm.hist[(key[u] >> shift) & ((1u << bits) - 1u)], 1u);
            }
          }
        }
        __syncthreads();
        uint32_t* total = sm.hist;
        if (sliced) {
          total = sm.total[pass & 1];
          const uint32_t at = peer_addr(smem_u32(total), 0);
          const uint4 four = *reinterpret_cast<const uint4*>(&sm.hist[kMine * threadIdx.x]);
          const uint32_t mine = at + 4 * kMine * threadIdx.x;
          if (four.x) add_cluster(mine, four.x);
          if (four.y) add_cluster(mine + 4, four.y);
          if (four.z) add_cluster(mine + 8, four.z);
          if (four.w) add_cluster(mine + 12, four.w);
          clear(sm.total[(pass + 1) & 1]);  // read in the pass before, added to in the next
          cluster_sync();
        }
        if (!sliced || rank == 0) {
          // Thread i has kMine bins counted from the top, so that scans run from the largest
          // key down.
          const int top = kBins - 1 - kMine * static_cast<int>(threadIdx.x);
          const uint4 four = *reinterpret_cast<const uint4*>(&total[top - 3]);
          const uint32_t mine = four.x + four.y + four.z + four.w;
          uint32_t all;
          uint32_t upto = scan_before(mine, sm.warp_sum, all);
          if (upto < want && want <= upto + mine) {
            int e = 0;
            for (; want > upto + total[top - e]; ++e) upto += total[top - e];
            sm.found[0] = top - e;
            sm.found[1] = want - upto;
            for (int r = 1; sliced && r < ranks; ++r) {
              st_cluster(peer_addr(smem_u32(&sm.found[0]), r), top - e);
              st_cluster(peer_addr(smem_u32(&sm.found[1]), r), want - upto);
            }
          }
        }
        sync();  // `found` is written, and the histograms are read
        threshold = (threshold << bits) | sm.found[0];
        want = sm.found[1];
      }
    } else {
      __syncthreads();  // the keys are written
    }
    // Kept: sinks, recent, keys above the threshold, and the first `want` equal to it.
    auto state = [&](int j, uint32_t key) {  // 1: kept for sure, 2: equal to the threshold
      if (j < a.sinks || j >= late) return 1;
      return none ? 0 : key > threshold ? 1 : key == threshold ? 2 : 0;
    };
    // Slots in order: each warp takes a run of the chunk, notes for each 32 entries which are
    // kept and counts them; after one scan it walks its notes.
    uint32_t sure_before = 0, equal_before = 0;  // of the entries before the chunk
    uint32_t before, all;                        // both counts, 16 bits each: before the run, of the chunk
    int run;                                     // groups of 32 of a warp
    auto note = [&](int base) {
      const int count = min(hi - base, kChunk);
      run = (count + 32 * kWarps - 1) / (32 * kWarps);
      uint32_t mine = 0;
      for (int g0 = wid * run; g0 < (wid + 1) * run && 32 * g0 < count; g0 += kAhead) {
        int st[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = 32 * (g0 + u) + lane;
          st[u] = g0 + u < (wid + 1) * run && i < count ? state(base + i, sm.key[i]) : 0;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const uint2 bits = make_uint2(__ballot_sync(0xffffffffu, st[u] == 1), __ballot_sync(0xffffffffu, st[u] == 2));
          if (lane == 0 && g0 + u < (wid + 1) * run && 32 * (g0 + u) < count) sm.ballot[g0 + u] = bits;
          mine += __popc(bits.x) | (__popc(bits.y) << 16);
        }
      }
      before = __shfl_sync(0xffffffffu, scan_before(lane == 0 ? mine : 0u, sm.warp_sum, all), 0);
    };
    auto emit = [&](int base) {
      const int count = min(hi - base, kChunk);
      uint32_t s = sure_before + (before & 0xffffu), e = equal_before + (before >> 16);
      const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
      for (int g = wid * run; g < min((wid + 1) * run, (count + 31) / 32); ++g) {
        const uint2 bits = sm.ballot[g];
        const uint32_t equal_at = e + __popc(bits.y & below);
        const int slot = static_cast<int>(s + __popc(bits.x & below) + min(equal_at, want));
        const bool keeps = ((bits.x >> lane) & 1u) || (((bits.y >> lane) & 1u) && equal_at < want);
        if (keeps && (sliced || (slot >= slot0 && slot < slot1))) {
          const int j = base + 32 * g + lane;
          index[slot] = j;
          if (!sliced) sm.list[slot - slot0] = static_cast<uint16_t>(j);
        }
        s += __popc(bits.x);
        e += __popc(bits.y);
      }
      sure_before += all & 0xffffu;
      equal_before += all >> 16;
    };
    if (once) {
      note(lo);
    } else {
      uint32_t sure = 0, equal = 0;
      for (int base = lo; base < hi; base += kChunk) {
        load(base);
        for (int j = base + threadIdx.x; j < min(hi, base + kChunk); j += kThreads) {
          const int st = state(j, sm.key[j - base]);
          sure += st == 1;
          equal += st == 2;
        }
      }
      scan_before(sure, sm.warp_sum, before);
      scan_before(equal, sm.warp_sum, all);
    }
    if (sliced) {
      if (threadIdx.x == 0) {
        sm.counts[0] = once ? all & 0xffffu : before;
        sm.counts[1] = once ? all >> 16 : all;
      }
      cluster_sync();
      for (int r = 0; r < rank; ++r) {
        const uint4 y = ld_cluster_v4(peer_addr(smem_u32(sm.counts), r));
        sure_before += y.x;
        equal_before += y.y;
      }
    }
    if (once) {
      emit(lo);
    } else {
      for (int base = lo; base < hi; base += kChunk) {
        __syncthreads();  // the keys and notes of the chunk before have been read
        load(base);
        __syncthreads();
        note(base);
        emit(base);
      }
    }
    sync();  // the whole index (the share's list) is written; no CTA reads another's memory any more
  }

  // Copy slots [slot0, slot1).
  using T = typename Piece<VEC>::T;
  const int pieces = a.D / VEC;
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + h * a.k_stride[2];
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
  uint16_t* ko = static_cast<uint16_t*>(a.k_out) + b * a.k_out_stride[0] + h * a.k_out_stride[2];
  uint16_t* vo = static_cast<uint16_t*>(a.v_out) + b * a.v_out_stride[0] + h * a.v_out_stride[2];
  auto from_of = [&](int slot) { return n <= a.keep ? slot : sliced ? index[slot] : sm.list[slot - slot0]; };
  // Weights by themselves: beside the rows they cost registers, and the spills' traffic was 3%.
  for (int s0 = slot0 + threadIdx.x; s0 < slot1; s0 += kThreads * kAhead) {
    int from[kAhead];
    float wt[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int slot = s0 + u * kThreads;
      from[u] = slot < min(slot1, kept) ? from_of(slot) : -1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) wt[u] = from[u] < 0 ? 0.f : __ldcg(w + from[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int slot = s0 + u * kThreads;
      if (slot >= slot1) break;
      w_out[slot] = wt[u];
      if (n <= a.keep) index[slot] = from[u];
    }
  }
  const int all = (slot1 - slot0) * pieces;
  for (int i0 = threadIdx.x; i0 < all; i0 += kThreads * kRowsInFlight) {
    T x[kRowsInFlight], y[kRowsInFlight];
    int slot[kRowsInFlight], from[kRowsInFlight], c[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      const int i = i0 + u * kThreads, s = i / pieces;
      slot[u] = i < all ? slot0 + s : -1;
      c[u] = (i - s * pieces) * VEC;
      from[u] = slot[u] < 0 || slot[u] >= kept ? -1 : from_of(slot[u]);
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      x[u] = y[u] = Piece<VEC>::zero();
      if (from[u] >= 0) {
        x[u] = __ldcg(reinterpret_cast<const T*>(k + from[u] * a.k_stride[1] + c[u]));
        y[u] = __ldcg(reinterpret_cast<const T*>(v + from[u] * a.v_stride[1] + c[u]));
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      if (slot[u] < 0) continue;
      *reinterpret_cast<T*>(ko + slot[u] * a.k_out_stride[1] + c[u]) = x[u];
      *reinterpret_cast<T*>(vo + slot[u] * a.v_out_stride[1] + c[u]) = y[u];
    }
  }
}

template <int VEC>
cudaError_t launch_evict_t(const fa4d_evict_args& a, int ranks, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(evict_kernel<VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem));
  if (e != cudaSuccess) return e;
  return launch_chained(evict_kernel<VEC>, dim3(static_cast<unsigned>(ranks) * a.B * a.Hk), kThreads, sizeof(Smem), ranks, s, a);
}

}  // namespace

cudaError_t launch_evict(const fa4d_evict_args& a, bool vec, int sms, cudaStream_t s) {
  // CTAs per (request, KV head): the fewest that give every SM one, at most 8 (B32 Hk8, 2304
  // slots to 1536: 75.5 us with 1, 79 with 2, 104 with 8; B4 Hk8, 65536 to 32768: 484 with 1,
  // 164 with 4, 119 with 8).
  int ranks = 1;
  while (ranks < 8 && static_cast<int64_t>(a.B) * a.Hk * ranks < sms) ranks *= 2;
  return vec ? launch_evict_t<8>(a, ranks, s) : launch_evict_t<1>(a, ranks, s);
}

}  // namespace fa4d
