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
constexpr int kBins = 2048;  // of a radix pass: 11, 11 and 10 bits of the weight
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
  alignas(16) uint32_t counts[4];  // of this CTA's slice: kept for sure, equal to the threshold
  uint32_t warp_sum[2][kWarps];
  uint32_t found[2];
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

template <int VEC>
__global__ void __launch_bounds__(kThreads) evict_kernel(const __grid_constant__ fa4d_evict_args a) {
  __shared__ Smem sm;
  const int rank = static_cast<int>(cluster_rank()), ranks = static_cast<int>(cluster_size());
  const int item = static_cast<int>(blockIdx.x) / ranks;
  const int b = item / a.Hk, h = item - b * a.Hk;
  const int n = min(max(__ldg(a.lengths + b), 0), a.C);
  const int kept = min(n, a.keep);
  const float* w = a.weights + b * a.weights_stride[0] + h * a.weights_stride[1];
  float* w_out = a.weights_out + b * a.weights_out_stride[0] + h * a.weights_out_stride[1];
  int32_t* index = a.index_out + static_cast<int64_t>(item) * a.keep;
  if (h == 0 && rank == 0 && threadIdx.x == 0) a.lengths_out[b] = kept;

  if (n > a.keep) {
    // The middle [a.sinks, late) gives its `want` heaviest entries.
    const int late = n - a.recent;
    const uint32_t want_all = a.keep - a.sinks - a.recent;
    const int per = (n + ranks - 1) / ranks;
    const int lo = min(rank * per, n), hi = min(lo + per, n);
    const int mid_lo = max(lo, a.sinks), mid_hi = min(hi, late);

    // Radix selection of the want_all-th largest key of the middle.
    uint32_t want = want_all, prefix = 0;
    if (want_all > 0) {
      constexpr int kShift[3] = {21, 10, 0};
      constexpr int kBits[3] = {11, 11, 10};
#pragma unroll
      for (int pass = 0; pass < 3; ++pass) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sm.hist[i] = 0;
        __syncthreads();
        for (int j = mid_lo + threadIdx.x; j < mid_hi; j += kThreads) {
          const uint32_t key = order_key(__ldg(w + j));
          if (pass == 0 || (key >> (kShift[pass] + kBits[pass])) == prefix)
            atomicAdd(&sm.hist[(key >> kShift[pass]) & ((1u << kBits[pass]) - 1u)], 1u);
        }
        cluster_sync();
        // Thread i has bins 4 i' .. 4 i' + 3 with i' counted from the top, so that scans run
        // from the largest key down.
        const int bin0 = kBins - 4 - 4 * threadIdx.x;
        uint4 c = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t mine = smem_u32(&sm.hist[bin0]);
        for (int r = 0; r < ranks; ++r) {
          const uint4 x = ld_cluster_v4(peer_addr(mine, r));
          c.x += x.x;
          c.y += x.y;
          c.z += x.z;
          c.w += x.w;
        }
        uint32_t all;
        const uint32_t above = scan_before(c.x + c.y + c.z + c.w, sm.warp_sum[0], all);
        const uint32_t cnt[4] = {c.w, c.z, c.y, c.x};
        uint32_t upto = above;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (upto < want && want <= upto + cnt[e]) {
            sm.found[0] = bin0 + 3 - e;
            sm.found[1] = want - upto;
          }
          upto += cnt[e];
        }
        cluster_sync();  // every CTA has read the histograms; `found` is written
        prefix = (prefix << kBits[pass]) | sm.found[0];
        want = sm.found[1];
      }
    }
    // Kept: sinks, recent, keys above `prefix`, and the first `want` equal to it.
    const bool none = want_all == 0;
    auto state = [&](int j, float& x) {  // 1: kept for sure, 2: equal to the threshold
      x = __ldg(w + j);
      if (j < a.sinks || j >= late) return 1;
      const uint32_t key = order_key(x);
      return none ? 0 : key > prefix ? 1 : key == prefix ? 2 : 0;
    };
    uint32_t sure = 0, equal = 0;
    for (int j = lo + threadIdx.x; j < hi; j += kThreads) {
      float x;
      const int st = state(j, x);
      sure += st == 1;
      equal += st == 2;
    }
    uint32_t sure_all, equal_all;
    scan_before(sure, sm.warp_sum[0], sure_all);
    scan_before(equal, sm.warp_sum[1], equal_all);
    if (threadIdx.x == 0) {
      sm.counts[0] = sure_all;
      sm.counts[1] = equal_all;
    }
    cluster_sync();
    uint32_t sure_before = 0, equal_before = 0;  // of the entries before this chunk
    for (int r = 0; r < rank; ++r) {
      const uint4 x = ld_cluster_v4(peer_addr(smem_u32(sm.counts), r));
      sure_before += x.x;
      equal_before += x.y;
    }
    for (int j0 = lo; j0 < hi; j0 += kThreads) {
      const int j = j0 + threadIdx.x;
      float x = 0.f;
      const int st = j < hi ? state(j, x) : 0;
      uint32_t chunk;  // both counts in one scan: at most 512 each
      const uint32_t before = scan_before((st == 1 ? 1u : 0u) | (st == 2 ? 0x10000u : 0u), sm.warp_sum[0], chunk);
      const uint32_t s = sure_before + (before & 0xffffu), e = equal_before + (before >> 16);
      if (st == 1 || (st == 2 && e < want)) {
        const uint32_t slot = s + min(e, want);
        index[slot] = j;
        w_out[slot] = x;
      }
      sure_before += chunk & 0xffffu;
      equal_before += chunk >> 16;
    }
    cluster_sync();  // the whole index is written, and no CTA reads another's memory any more
  }

  // Copy slots [slot0, slot1).
  const int share = (a.keep + ranks - 1) / ranks;
  const int slot0 = min(rank * share, a.keep), slot1 = min(slot0 + share, a.keep);
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
      from[u] = slot[u] < 0 || slot[u] >= kept ? -1 : n > a.keep ? index[slot[u]] : slot[u];
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
