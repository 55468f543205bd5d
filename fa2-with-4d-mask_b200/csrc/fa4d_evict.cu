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
#include "fa4d_ptx.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kEach = 16;                    // weights of a thread, kept in registers
constexpr int kChunk = kThreads * kEach;     // weights of a CTA at a time
constexpr int kBins = 2048;                  // of a radix pass: 11, 11 and 10 bits of the weight
constexpr int kRowsInFlight = 4;

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
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

struct Smem {
  alignas(16) uint32_t hist[kBins];
  alignas(16) uint32_t counts[4];     // of this CTA's slice: kept for sure, equal to the threshold
  uint32_t group[kEach * kWarps];     // of each 32 weights in order: both counts, 16 bits each
  uint32_t warp_sum[kWarps];
  uint32_t found[2];
  int32_t list[kChunk];               // slots of this CTA's share (selection without slices)
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
// each CTA takes a slice of the weights.  Weights stay in registers across the passes
// (re-read where a slice is longer than kChunk).
template <int VEC>
__global__ void __launch_bounds__(kThreads, 2) evict_kernel(const __grid_constant__ fa4d_evict_args a) {
  __shared__ Smem sm;
  const int rank = static_cast<int>(cluster_rank()), ranks = static_cast<int>(cluster_size());
  const int item = static_cast<int>(blockIdx.x) / ranks;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int b = item / a.Hk, h = item - b * a.Hk;
  const int n = min(max(__ldg(a.lengths + b), 0), a.C);
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
    uint32_t want = a.keep - a.sinks - a.recent, prefix = 0;
    const bool none = want == 0;
    const int per = sliced ? (n + ranks - 1) / ranks : n;
    const int lo = sliced ? min(rank * per, n) : 0, hi = min(lo + per, n);
    const bool once = hi - lo <= kChunk;

    float x[kEach];  // the weights j = base + i * kThreads + threadIdx.x
    auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int j = base + i * kThreads + threadIdx.x;
        x[i] = j < hi ? __ldg(w + j) : 0.f;
      }
    };
    auto in_middle = [&](int j) { return j >= a.sinks && j < late && j < hi; };
    load(lo);

    // Radix selection of the want-th largest key of the middle, from the top bits down.
    if (!none) {
      constexpr int kShift[3] = {21, 10, 0};
      constexpr int kBits[3] = {11, 11, 10};
#pragma unroll
      for (int pass = 0; pass < 3; ++pass) {
        *reinterpret_cast<uint4*>(&sm.hist[4 * threadIdx.x]) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        for (int base = lo; base < hi; base += kChunk) {
          if (!once) load(base);
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            const uint32_t key = order_key(x[i]);
            if (in_middle(base + i * kThreads + threadIdx.x) &&
                (pass == 0 || (key >> (kShift[pass] + kBits[pass])) == prefix))
              atomicAdd(&sm.hist[(key >> kShift[pass]) & ((1u << kBits[pass]) - 1u)], 1u);
          }
        }
        // Thread i has four bins, counted from the top, so that scans run from the largest
        // key down.
        const int bin0 = kBins - 4 - 4 * threadIdx.x;
        uint4 c = make_uint4(0u, 0u, 0u, 0u);
        if (sliced) {
          cluster_sync();
          const uint32_t mine = smem_u32(&sm.hist[bin0]);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r >= ranks) break;
            const uint4 y = ld_cluster_v4(peer_addr(mine, r));
            c.x += y.x;
            c.y += y.y;
            c.z += y.z;
            c.w += y.w;
          }
        } else {
          __syncthreads();
          c = *reinterpret_cast<const uint4*>(&sm.hist[bin0]);
        }
        uint32_t all;
        uint32_t upto = scan_before(c.x + c.y + c.z + c.w, sm.warp_sum, all);
        const uint32_t cnt[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (upto < want && want <= upto + cnt[e]) {
            sm.found[0] = bin0 + 3 - e;
            sm.found[1] = want - upto;
          }
          upto += cnt[e];
        }
        // `found` is written, and the histograms are read.
        if (sliced)
          cluster_sync();
        else
          __syncthreads();
        prefix = (prefix << kBits[pass]) | sm.found[0];
        want = sm.found[1];
      }
    }
    // Kept: sinks, recent, keys above `prefix`, and the first `want` equal to it.
    auto state = [&](int j, float v) {  // 1: kept for sure, 2: equal to the threshold
      if (j >= hi) return 0;
      if (j < a.sinks || j >= late) return 1;
      const uint32_t key = order_key(v);
      return none ? 0 : key > prefix ? 1 : key == prefix ? 2 : 0;
    };
    uint32_t sure_before = 0, equal_before = 0;  // of the entries before the chunk
    if (sliced) {
      uint32_t sure = 0, equal = 0;
      for (int base = lo; base < hi; base += kChunk) {
        if (!once) load(base);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int st = state(base + i * kThreads + threadIdx.x, x[i]);
          sure += st == 1;
          equal += st == 2;
        }
      }
      uint32_t sure_all, equal_all;
      scan_before(sure, sm.warp_sum, sure_all);
      scan_before(equal, sm.warp_sum, equal_all);
      if (threadIdx.x == 0) {
        sm.counts[0] = sure_all;
        sm.counts[1] = equal_all;
      }
      cluster_sync();
      for (int r = 0; r < rank; ++r) {
        const uint4 y = ld_cluster_v4(peer_addr(smem_u32(sm.counts), r));
        sure_before += y.x;
        equal_before += y.y;
      }
    }
    // Slots in order: a warp's 32 weights of each i by ballots, the groups by one scan.
    for (int base = lo; base < hi; base += kChunk) {
      if (!once) load(base);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int st = state(base + i * kThreads + threadIdx.x, x[i]);
        const uint32_t sure = __ballot_sync(0xffffffffu, st == 1), equal = __ballot_sync(0xffffffffu, st == 2);
        if (lane == 0) sm.group[i * kWarps + wid] = __popc(sure) | (__popc(equal) << 16);
      }
      __syncthreads();
      uint32_t all;  // at most kChunk in each half
      const uint32_t before =
          scan_before(threadIdx.x < kEach * kWarps ? sm.group[threadIdx.x] : 0u, sm.warp_sum, all);
      if (threadIdx.x < kEach * kWarps) sm.group[threadIdx.x] = before;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int j = base + i * kThreads + threadIdx.x;
        const int st = state(j, x[i]);
        const uint32_t sure = __ballot_sync(0xffffffffu, st == 1), equal = __ballot_sync(0xffffffffu, st == 2);
        const uint32_t below = (1u << lane) - 1u, group = sm.group[i * kWarps + wid];
        const uint32_t s = sure_before + (group & 0xffffu) + __popc(sure & below);
        const uint32_t e = equal_before + (group >> 16) + __popc(equal & below);
        if (st == 1 || (st == 2 && e < want)) {
          const int slot = static_cast<int>(s + min(e, want));
          if (sliced || (slot >= slot0 && slot < slot1)) {
            index[slot] = j;
            w_out[slot] = x[i];
            if (!sliced) sm.list[slot - slot0] = j;
          }
        }
      }
      sure_before += all & 0xffffu;
      equal_before += all >> 16;
      if (!once) __syncthreads();  // the groups have been read
    }
    // The whole index (the share's list) is written; no CTA reads another's memory any more.
    if (sliced)
      cluster_sync();
    else
      __syncthreads();
  }

  // Copy slots [slot0, slot1).
  using T = typename Piece<VEC>::T;
  const int pieces = a.D / VEC;
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + h * a.k_stride[2];
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2];
  uint16_t* ko = static_cast<uint16_t*>(a.k_out) + b * a.k_out_stride[0] + h * a.k_out_stride[2];
  uint16_t* vo = static_cast<uint16_t*>(a.v_out) + b * a.v_out_stride[0] + h * a.v_out_stride[2];
  const int all = (slot1 - slot0) * pieces;
  for (int i0 = threadIdx.x; i0 < all; i0 += kThreads * kRowsInFlight) {
    T x[kRowsInFlight], y[kRowsInFlight];
    int slot[kRowsInFlight], from[kRowsInFlight], c[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      const int i = i0 + u * kThreads;
      const int s = i / pieces;
      slot[u] = i < all ? slot0 + s : -1;
      c[u] = (i - s * pieces) * VEC;
      from[u] = slot[u] < 0 || slot[u] >= kept ? -1 : n <= a.keep ? slot[u] : sliced ? index[slot[u]] : sm.list[s];
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      x[u] = y[u] = Piece<VEC>::zero();
      if (from[u] >= 0) {
        x[u] = __ldg(reinterpret_cast<const T*>(k + from[u] * a.k_stride[1] + c[u]));
        y[u] = __ldg(reinterpret_cast<const T*>(v + from[u] * a.v_stride[1] + c[u]));
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      if (slot[u] < 0) continue;
      *reinterpret_cast<T*>(ko + slot[u] * a.k_out_stride[1] + c[u]) = x[u];
      *reinterpret_cast<T*>(vo + slot[u] * a.v_out_stride[1] + c[u]) = y[u];
      if (c[u] == 0 && (n <= a.keep || from[u] < 0)) {  // where no selection wrote them
        index[slot[u]] = from[u];
        w_out[slot[u]] = from[u] < 0 ? 0.f : __ldg(w + from[u]);
      }
    }
  }
}

template <int VEC>
cudaError_t launch_evict_t(const fa4d_evict_args& a, int ranks, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ranks) * a.B * a.Hk);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_kernel<VEC>, a);
}

}  // namespace

cudaError_t launch_evict(const fa4d_evict_args& a, bool vec, int sms, cudaStream_t s) {
  // CTAs per (request, KV head): the fewest that give every SM two, at most 8.
  int ranks = 1;
  while (ranks < 8 && static_cast<int64_t>(a.B) * a.Hk * ranks < 2LL * sms) ranks *= 2;
  return vec ? launch_evict_t<8>(a, ranks, s) : launch_evict_t<1>(a, ranks, s);
}

}  // namespace fa4d
