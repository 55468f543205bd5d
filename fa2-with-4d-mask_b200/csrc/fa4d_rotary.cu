// fa4d_rotary.cu — rotary positions with several axes: the training form (q and k turned,
// or turned back for the gradient) and the serving form that also appends to a cache.
//
// Pair i of a head is multiplied, as a complex number, by e^(i phi) with
// phi = position(axis of i) * theta_i.  The angle is kept as a fraction of a turn in 64-bit
// fixed point: position * turn_i modulo 2^64 is exact, so what a position adds to the error is
// its multiple of turn_i's own rounding, about 2^-64 turns (a 32-bit product of position and
// frequency is off by 4e-3 rad at position 65536), and the fraction's top 32 bits go to sincospif,
// whose argument, rounded to 2^-25 turns, then needs no range reduction.
//
// Bound by memory: each element is read once and written once.
#include "fa4d.h"
#include "fa4d_kernels.h"
#include "fa4d_launch.cuh"
#include "fa4d_rotary.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 128;

// One thread: one chunk of a token, for a range of the q and k heads, so the angles are
// computed once for kHeads heads and more; the loads of kHeads heads are in flight together.
// Measured, one direction: B4 T8192 Hq32 Hk8 D128 104.6 us (6.4 TB/s, the measured copy rate),
// B1 31.2 us (5.4 TB/s), B2 T16385 Hq16 Hk8 D256 129 us (6.2 TB/s; 139 with the angles worked out
// before the first loads).  Two heads at a time took 135 us there, eight the same as four.
constexpr int kHeads = 4;

template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ fa4d_rotary_args a, int chunks,
                                                          int heads_each) {
  pdl_wait();
  pdl_launch();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t n = id / chunks;
  if (n >= static_cast<int64_t>(a.B) * a.T) return;
  const int c = static_cast<int>(id - n * chunks);
  const int64_t b = n / a.T, t = n - b * a.T;
  Chunk<VEC, kAdj> ch(a.table, c);

  const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1];
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1];
  uint16_t* qo = static_cast<uint16_t*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1];
  uint16_t* ko = static_cast<uint16_t*>(a.k_out) + b * a.k_out_stride[0] + t * a.k_out_stride[1];
  const int first = blockIdx.y * heads_each, end = min(first + heads_each, a.Hq + a.Hk);
  for (int h0 = first; h0 < end; h0 += kHeads) {
    typename Run<VEC>::T x[kHeads], y[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u;
      if (h >= end) break;
      const uint16_t* src = h < a.Hq ? q + h * a.q_stride[2] : k + (h - a.Hq) * a.k_stride[2];
      x[u] = Run<VEC>::load(src + ch.at0);
      y[u] = Run<VEC>::load(src + ch.at1);
    }
    // The angles, while the first heads are on their way.
    if (h0 == first) ch.turn_to(a.table, a.positions, a.positions_bits, a.positions_stride, b, t, c, a.inverse != 0);
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u;
      if (h >= end) break;
      if (!ch.copied) turn<kBF16, kAdj>(x[u], y[u], ch.cs, ch.sn);
      uint16_t* dst = h < a.Hq ? qo + h * a.q_out_stride[2] : ko + (h - a.Hq) * a.k_out_stride[2];
      Run<VEC>::store(dst + ch.at0, x[u]);
      Run<VEC>::store(dst + ch.at1, y[u]);
    }
  }
}

// One thread: one chunk of one head (q, k or v) of a new token.  A decode step has few
// tokens, so everything is spread over threads and the angles are computed per head; latency
// bounds it (one token 3.5 us, 160 tokens 5.0 us, back to back).
template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const __grid_constant__ fa4d_rotary_append_args a,
                                                                 int chunks, int* status) {
  pdl_wait();
  pdl_launch();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int heads = a.Hq + 2 * a.Hk;
  const int64_t row = id / chunks, n = row / heads;
  if (n >= static_cast<int64_t>(a.B) * a.T) return;
  const int c = static_cast<int>(id - row * chunks);
  const int h = static_cast<int>(row - n * heads);
  const int64_t b = n / a.T, t = n - b * a.T;
  const int64_t had = max(__ldcg(a.lengths + b), 0);
  if (h == 0 && c == 0 && t == 0)
    a.lengths_out[b] = static_cast<int32_t>(min(had + a.T, static_cast<int64_t>(a.C)));

  const int64_t slot = had + t;
  const bool fits = slot < a.C;
  if (h >= a.Hq && !fits) {
    if (h == a.Hq && c == 0) atomicOr(status, FA4D_DEV_CACHE_FULL);
    return;
  }
  Chunk<VEC, kAdj> ch(a.table, c);
  const uint16_t* src;
  uint16_t* dst;
  if (h < a.Hq) {
    src = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2];
    dst = static_cast<uint16_t*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1] + h * a.q_out_stride[2];
  } else if (h < a.Hq + a.Hk) {
    const int hk = h - a.Hq;
    src = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1] + hk * a.k_stride[2];
    dst = static_cast<uint16_t*>(a.k_cache) + b * a.k_cache_stride[0] + slot * a.k_cache_stride[1] +
          hk * a.k_cache_stride[2];
  } else {
    const int hk = h - a.Hq - a.Hk;
    src = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + t * a.v_stride[1] + hk * a.v_stride[2];
    dst = static_cast<uint16_t*>(a.v_cache) + b * a.v_cache_stride[0] + slot * a.v_cache_stride[1] +
          hk * a.v_cache_stride[2];
    if (a.weights && c == 0) a.weights[b * a.weights_stride[0] + hk * a.weights_stride[1] + slot] = 0.f;
  }
  typename Run<VEC>::T x = Run<VEC>::load(src + ch.at0), y = Run<VEC>::load(src + ch.at1);
  if (!ch.copied && h < a.Hq + a.Hk) {
    ch.turn_to(a.table, a.positions, a.positions_bits, a.positions_stride, b, t, c, false);
    turn<kBF16, kAdj>(x, y, ch.cs, ch.sn);
  }
  Run<VEC>::store(dst + ch.at0, x);
  Run<VEC>::store(dst + ch.at1, y);
}

int chunks_of(const fa4d_rotary_table& tab, int vec) {
  return tab.rotary_dim / 2 / vec + (tab.D - tab.rotary_dim) / (2 * vec);
}

template <int VEC, bool kBF16>
cudaError_t launch_rotary_t(const fa4d_rotary_args& a, int sms, cudaStream_t s) {
  const int chunks = chunks_of(a.table, VEC), heads = a.Hq + a.Hk;
  const int64_t threads = static_cast<int64_t>(a.B) * a.T * chunks;
  // Heads are split over the grid until about one full load of threads (2048 an SM) runs.
  const int64_t want = (static_cast<int64_t>(sms) * 2048 + threads - 1) / threads;
  const int split = static_cast<int>(min(want, static_cast<int64_t>((heads + kHeads - 1) / kHeads)));
  const int each = (heads + split - 1) / split;
  const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads), (heads + each - 1) / each);
  auto kern = a.table.pairing == FA4D_PAIR_ADJACENT ? rotary_kernel<kBF16, true, VEC> : rotary_kernel<kBF16, false, VEC>;
  return launch_chained(kern, grid, kThreads, 0, 1, s, a, chunks, each);
}

template <int VEC, bool kBF16>
cudaError_t launch_append_t(const fa4d_rotary_append_args& a, int* status, cudaStream_t s) {
  const int chunks = chunks_of(a.table, VEC);
  const int64_t threads = static_cast<int64_t>(a.B) * a.T * (a.Hq + 2 * a.Hk) * chunks;
  const unsigned grid = static_cast<unsigned>((threads + kThreads - 1) / kThreads);
  auto kern =
      a.table.pairing == FA4D_PAIR_ADJACENT ? rotary_append_kernel<kBF16, true, VEC> : rotary_append_kernel<kBF16, false, VEC>;
  return launch_chained(kern, dim3(grid), kThreads, 0, 1, s, a, chunks, status);
}

}  // namespace

cudaError_t launch_rotary(const fa4d_rotary_args& a, bool vec, int sms, cudaStream_t s) {
  const bool bf16 = a.dtype == FA4D_BF16;
  if (vec) return bf16 ? launch_rotary_t<8, true>(a, sms, s) : launch_rotary_t<8, false>(a, sms, s);
  return bf16 ? launch_rotary_t<1, true>(a, sms, s) : launch_rotary_t<1, false>(a, sms, s);
}

cudaError_t launch_rotary_append(const fa4d_rotary_append_args& a, bool vec, int* status, cudaStream_t s) {
  const bool bf16 = a.dtype == FA4D_BF16;
  if (vec) return bf16 ? launch_append_t<8, true>(a, status, s) : launch_append_t<8, false>(a, status, s);
  return bf16 ? launch_append_t<1, true>(a, status, s) : launch_append_t<1, false>(a, status, s);
}

}  // namespace fa4d
