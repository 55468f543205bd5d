// fa4d_norm.cu — training form of the norm of each head with the rotary turn in the same pass, and
// its gradient.
//
// Of a head x[D] with weights w: r = (mean x^2 + eps)^-1/2, y = turn(x r w).  Of dy, with
// g = turn^-1(dy):  dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x)).
// The backward pass works r out again from x, which it reads in any case.
//
// The forward reads and writes each element once, the backward reads x and dy and writes dx, which bounds
// long inputs.  Measured, forward and backward: B2 T16385 Hq16 Hk8 D256 fp16 130 and 205 us (805 and 1208
// MB: 6.2 and 5.9 TB/s, 95% and 90% of the measured copy rate).  B1 T8192 Hq32 Hk8 D128 bf16 33 and 49 us
// (168 and 252 MB: 5.1 TB/s, 78%): there the division bounds it, 512 groups of tokens over 296 blocks of
// q in two rounds, the second 73% full.
#include <algorithm>

#include "fa4d.h"
#include "fa4d_kernels.h"
#include "fa4d_launch.cuh"
#include "fa4d_norm.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 128;

// Blocks of an SM, and ranges of at most so many heads (their angles are worked out once).  The grid
// fills the GPU once; with many tokens it is kWaves times as large, which evens out what the SMs are
// apart (B2 T16385 Hq16 Hk8 D256: forward 150 us once, 130 three times; B1 T8192 Hq32 Hk8 D128, whose
// blocks have two rounds, 34 and 35; backward 204 and 192, 49 and 57).
constexpr int kFwdPerSm = 5, kBwdPerSm = 3, kHeadsEach = 16;
constexpr int kFwdWaves = 3, kBwdWaves = 2;
constexpr int kLong = 8;  // rounds of a block

// The grid: `q_blocks` blocks for q, then those for k, in proportion to their heads; of each, `parts`
// ranges of heads side by side, and over those the tokens.
struct NormGrid {
  int lanes, chunks;
  int q_blocks, q_parts, q_each;
  int k_blocks, k_parts, k_each;
};

// A block's part.
struct Part {
  bool is_q;
  int first, end;      // heads
  uint32_t x, across;  // which of so many blocks that share the tokens
  __device__ __forceinline__ Part(const NormGrid& g, int Hq, int Hk) {
    is_q = blockIdx.x < g.q_blocks;
    const int id = is_q ? blockIdx.x : blockIdx.x - g.q_blocks, parts = is_q ? g.q_parts : g.k_parts;
    const int each = is_q ? g.q_each : g.k_each;
    first = id % parts * each;
    end = min(first + each, is_q ? Hq : Hk);
    x = id / parts;
    across = (is_q ? g.q_blocks : g.k_blocks) / parts;
  }
};

// One thread: a lane of a token's rows, for a range of q's or of k's heads (angles serve them all),
// token after token, `across` blocks apart.  What it reads comes into places of its own in shared
// memory, kDepth rows ahead (no barrier between threads): with loads into registers, four rows at a
// time, a warp had none on their way while it computed.  Forward and backward together, B2 T16385
// Hq16 Hk8 D256: 721 us with weights and turns read from memory and parameters by every thread, 431
// with those in shared memory, 340 with rows fed ahead, packed arithmetic and neighbouring 16 bytes
// a lane.
constexpr int kFwdDepth = 6, kBwdDepth = 4;
template <int VEC, bool kAdj, int kStreams, int kDepth>
class Feed {
 public:
  static constexpr int kBytes = VEC == 8 ? kDepth * kStreams * 2 * 16 * kThreads : 0;

  __device__ __forceinline__ Feed(uint8_t* smem, const RowLane<VEC, kAdj>& at_, const fa4d_rotary_args& a, uint32_t first_token,
                                  uint32_t step_, int first_, int end_)
      : at(at_), ring(reinterpret_cast<uint4*>(smem) + threadIdx.x), n(first_token), step(step_), tokens(a.B * static_cast<uint32_t>(a.T)),
        T(a.T), h(first_), first(first_), end(end_) {}
  __device__ __forceinline__ void add(int s, const void* base, const int64_t (&stride)[3]) {
    all[s] = static_cast<const uint16_t*>(base) + first * stride[2];
    batch[s] = stride[0];
    seq[s] = stride[1];
    head[s] = stride[2];
  }
  __device__ __forceinline__ void start() {
    place();
    if constexpr (VEC == 8)
#pragma unroll
      for (int i = 0; i < kDepth; ++i) bring(i);
  }
  // The row at `stage` (they come round in order), all streams.
  __device__ __forceinline__ void take(int stage, Raw<VEC> (&r)[kStreams]) {
    if constexpr (VEC == 8) {
      cp_async_wait<kDepth - 1>();
#pragma unroll
      for (int s = 0; s < kStreams; ++s) {
        const uint4* p = ring + (stage * kStreams + s) * 2 * kThreads;
        r[s].x[0] = at.live ? p[0] : make_uint4(0, 0, 0, 0);
        r[s].y[0] = at.live ? p[kThreads] : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int s = 0; s < kStreams; ++s)
        if (n < tokens) at.load(src[s], r[s]);
    }
  }
  // After the last use of what take() gave.
  __device__ __forceinline__ void next(int stage) {
    if constexpr (VEC == 8)
      bring(stage);
    else
      advance();
  }

 private:
  const RowLane<VEC, kAdj>& at;
  uint4* ring;  // [kDepth][kStreams][2], kThreads apart
  uint32_t n, step, tokens, T;
  int h, first, end;
  const uint16_t* all[kStreams];
  const uint16_t* src[kStreams];
  int64_t batch[kStreams], seq[kStreams], head[kStreams];

  __device__ __forceinline__ void place() {
    const uint32_t b = n / T, t = n - b * T;
#pragma unroll
    for (int s = 0; s < kStreams; ++s) src[s] = all[s] + b * batch[s] + t * seq[s];
  }
  __device__ __forceinline__ void advance() {
    if (++h < end) {
#pragma unroll
      for (int s = 0; s < kStreams; ++s) src[s] += head[s];
      return;
    }
    h = first;
    n += step;
    place();
  }
  __device__ __forceinline__ void bring(int stage) {
    if (at.live && n < tokens) {
#pragma unroll
      for (int s = 0; s < kStreams; ++s) {
        uint4* p = ring + (stage * kStreams + s) * 2 * kThreads;
        cp_async16(p, src[s] + at.at0[0], 16);
        cp_async16(p + kThreads, src[s] + at.at1[0], 16);
      }
    }
    cp_async_commit();
    advance();
  }
};

// The rows that a thread goes through: `live` ones of tokens (b, t), heads from `first` on.
struct Rows {
  uint32_t n, step;
  int iterations;
  __device__ __forceinline__ Rows(const fa4d_rotary_args& a, int lanes, const Part& part) {
    const uint32_t rows = kThreads / lanes, tokens = a.B * static_cast<uint32_t>(a.T), n0 = part.x * rows;
    step = part.across * rows;
    n = n0 + threadIdx.x / lanes;
    iterations = static_cast<int>((tokens - n0 + step - 1) / step) * (part.end - part.first);  // the same for all threads
  }
};

template <bool kBF16, bool kAdj, int VEC, int kLanes>
__global__ void __launch_bounds__(kThreads, kFwdPerSm) norm_rotary_kernel(
    const __grid_constant__ fa4d_norm_rotary_args args, const __grid_constant__ NormGrid grid) {
  const int lanes = kLanes ? kLanes : grid.lanes;
  using F = Feed<VEC, kAdj, 1, kFwdDepth>;
  extern __shared__ uint4 ring4[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(ring4);  // [F::kBytes]
  __shared__ Turns<VEC> turns;
  __shared__ Weights<VEC> weights;
  const fa4d_rotary_args& a = args.rotary;
  turns.template fill<kAdj>(a.table);
  const int lane = threadIdx.x & (lanes - 1);
  const Part heads(grid, a.Hq, a.Hk);
  const RowLane<VEC, kAdj> at(a.table, lane, grid.chunks);
  Rows rows(a, lanes, heads);
  F feed(ring, at, a, rows.n, rows.step, heads.first, heads.end);
  pdl_wait();
  pdl_launch();
  if (heads.is_q)
    feed.add(0, a.q, a.q_stride);
  else
    feed.add(0, a.k, a.k_stride);
  feed.start();
  weights.template fill<kBF16, kAdj>(a.table, heads.is_q ? args.norm.q_weight : args.norm.k_weight, args.norm.weight_f32 != 0);
  __syncthreads();
  const int64_t* so = heads.is_q ? a.q_out_stride : a.k_out_stride;
  const uint32_t tokens = a.B * static_cast<uint32_t>(a.T);
  const float mean = 1.f / a.table.D;
  uint16_t* dst = nullptr;
  bool live = false;
  Factors<VEC> factors;
  const bool copied = at.copied();
  int h = heads.first, stage = 0;
#pragma unroll 1
  for (int it = 0; it < rows.iterations; ++it) {
    Raw<VEC> raw[1];
    feed.take(stage, raw);
    if (h == heads.first) {
      live = rows.n < tokens;
      const uint32_t b = rows.n / a.T, t = rows.n - b * a.T;
      dst = static_cast<uint16_t*>(heads.is_q ? a.q_out : a.k_out) + b * so[0] + t * so[1] + h * so[2];
      if (live) {
        Turn<VEC> turn;
        at.angles(turns, a.positions, a.positions_bits, a.positions_stride, b, t, lane, turn);
        factors.set(turn);
        Pairs<VEC> w;
        at.weights(weights, lane, w);
        factors.weigh(w);
      }
    }
    Pairs<VEC> p;
    unpack_pairs<kBF16, kAdj>(raw[0], p);
    p.times(rsqrtf(row_sum<kLanes>(p.squares(), lanes) * mean + args.norm.eps));
    if (live) {
      factors.turn(p, copied);
      pack_pairs<kBF16, kAdj>(p, raw[0]);
      at.store(dst, raw[0]);
    }
    feed.next(stage);
    if (++stage == kFwdDepth) stage = 0;
    dst += so[2];
    if (++h == heads.end) {
      h = heads.first;
      rows.n += rows.step;
    }
  }
  if constexpr (VEC == 8) cp_async_wait_all();
}

// The gradient.  A thread adds the weights' gradient up over all its rows in registers, then the
// block over its threads in shared memory: one row of D sums a block, which weight_grad_kernel adds
// (always in the same order).
template <bool kBF16, bool kAdj, int VEC, int kLanes>
__global__ void __launch_bounds__(kThreads, kBwdPerSm) norm_rotary_grad_kernel(
    const __grid_constant__ fa4d_norm_rotary_bwd_args args, const __grid_constant__ NormGrid grid) {
  const int lanes = kLanes ? kLanes : grid.lanes;
  using F = Feed<VEC, kAdj, 2, kBwdDepth>;
  constexpr int P = kRowPairs<VEC> / 2;
  extern __shared__ uint4 ring4[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(ring4);  // [F::kBytes], and in the end the sums, [rows][D]
  __shared__ Turns<VEC> turns;
  __shared__ Weights<VEC> weights;
  const fa4d_rotary_args& a = args.rotary;
  turns.template fill<kAdj>(a.table);
  const int lane = threadIdx.x & (lanes - 1);
  const Part heads(grid, a.Hq, a.Hk);
  const RowLane<VEC, kAdj> at(a.table, lane, grid.chunks);
  Rows rows(a, lanes, heads);
  F feed(ring, at, a, rows.n, rows.step, heads.first, heads.end);
  pdl_wait();
  pdl_launch();
  if (heads.is_q) {
    feed.add(0, a.q, a.q_stride);
    feed.add(1, args.dq, args.dq_stride);
  } else {
    feed.add(0, a.k, a.k_stride);
    feed.add(1, args.dk, args.dk_stride);
  }
  feed.start();
  weights.template fill<kBF16, kAdj>(a.table, heads.is_q ? args.norm.q_weight : args.norm.k_weight, args.norm.weight_f32 != 0);
  __syncthreads();
  const int64_t* so = heads.is_q ? a.q_out_stride : a.k_out_stride;
  const uint32_t tokens = a.B * static_cast<uint32_t>(a.T);
  const float mean = 1.f / a.table.D;
  uint16_t* dx = nullptr;
  bool live = false;
  Turn<VEC> turn;
  const bool copied = at.copied();
  Pairs<VEC> dw;
#pragma unroll
  for (int j = 0; j < P; ++j) dw.a[j] = dw.b[j] = f2(0.f, 0.f);
  int h = heads.first, stage = 0;
#pragma unroll 1
  for (int it = 0; it < rows.iterations; ++it) {
    Raw<VEC> raw[2];
    feed.take(stage, raw);
    if (h == heads.first) {
      live = rows.n < tokens;
      const uint32_t b = rows.n / a.T, t = rows.n - b * a.T;
      dx = static_cast<uint16_t*>(heads.is_q ? a.q_out : a.k_out) + b * so[0] + t * so[1] + h * so[2];
      if (live) at.angles(turns, a.positions, a.positions_bits, a.positions_stride, b, t, lane, turn);
    }
    Pairs<VEC> x, d, g, w;
    unpack_pairs<kBF16, kAdj>(raw[0], x);
    unpack_pairs<kBF16, kAdj>(raw[1], d);
    at.weights(weights, lane, w);
    uint64_t dots = f2(0.f, 0.f);
    turn.back(d, g, copied);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      w.a[j] = fmul2(w.a[j], g.a[j]);
      w.b[j] = fmul2(w.b[j], g.b[j]);
      dots = ffma2(x.a[j], w.a[j], ffma2(x.b[j], w.b[j], dots));
    }
    const float2 both = f2_split(dots);
    const float square = row_sum<kLanes>(x.squares(), lanes), dot = row_sum<kLanes>(both.x + both.y, lanes);
    if (live) {
      // r times the dot product is of the gradient's size: r^2 alone passes fp32 beside the least epsilons.
      // Where the squares do (r = 0), the row's output is 0 whatever it holds, and so is its gradient.
      const float r = rsqrtf(square * mean + args.norm.eps), c = r > 0.f ? -(r * (r * (dot * mean))) : 0.f;
      const uint64_t rr = f2(r, r), cc = f2(c, c);
      x.times(r);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        dw.a[j] = ffma2(g.a[j], x.a[j], dw.a[j]);
        dw.b[j] = ffma2(g.b[j], x.b[j], dw.b[j]);
        g.a[j] = ffma2(x.a[j], cc, fmul2(w.a[j], rr));
        g.b[j] = ffma2(x.b[j], cc, fmul2(w.b[j], rr));
      }
      pack_pairs<kBF16, kAdj>(g, raw[0]);
      at.store(dx, raw[0]);
    }
    feed.next(stage);
    if (++stage == kBwdDepth) stage = 0;
    dx += so[2];
    if (++h == heads.end) {
      h = heads.first;
      rows.n += rows.step;
    }
  }
  if constexpr (VEC == 8) cp_async_wait_all();
  __syncthreads();
  // Over the block's rows.
  float* sums = reinterpret_cast<float*>(ring);
  const int row = threadIdx.x / lanes;
#pragma unroll
  for (int j = 0; j < 2 * P; ++j)
    if ((at.live >> (j / VEC)) & 1u) {
      const float2 u = f2_split(dw.a[j / 2]), v = f2_split(dw.b[j / 2]);
      const PairAt<VEC, kAdj> e(a.table, lane + 32 * (j / VEC), j % VEC);
      sums[row * a.table.D + e.e0] = j & 1 ? u.y : u.x;
      sums[row * a.table.D + e.e1] = j & 1 ? v.y : v.x;
    }
  __syncthreads();
  float* part = static_cast<float*>(args.workspace) + static_cast<int64_t>(blockIdx.x) * a.table.D;
  for (int e = threadIdx.x; e < a.table.D; e += kThreads) {
    float s = 0.f;
    for (int r = 0; r < kThreads / lanes; ++r) s += sums[r * a.table.D + e];
    part[e] = s;
  }
}

// Adds the blocks' rows: 8 columns a block, 32 threads each.
template <bool kBF16>
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* parts, int D, int q_rows, int k_rows, void* dwq, void* dwk,
                                                          bool f32) {
  __shared__ float sums[32][9];
  const bool is_q = blockIdx.y == 0;
  const int col = threadIdx.x & 7, at = threadIdx.x >> 3, e = blockIdx.x * 8 + col;
  const int rows = is_q ? q_rows : k_rows;
  pdl_wait();
  pdl_launch();
  const float* p = parts + (is_q ? 0 : static_cast<int64_t>(q_rows) * D);
  float s = 0.f;
  if (e < D)
#pragma unroll 8
    for (int r = at; r < rows; r += 32) s += __ldcg(p + static_cast<int64_t>(r) * D + e);
  sums[at][col] = s;
  __syncthreads();
  if (threadIdx.x < 8 && e < D) {
    float all = 0.f;
    for (int r = 0; r < 32; ++r) all += sums[r][threadIdx.x];
    void* dst = is_q ? dwq : dwk;
    if (f32)
      static_cast<float*>(dst)[e] = all;
    else
      static_cast<uint16_t*>(dst)[e] = to_h<kBF16>(all);
  }
}

NormGrid grid_of(const fa4d_rotary_args& a, int vec, int per_sm, int waves, int sms) {
  NormGrid g;
  g.lanes = row_lanes(a.table, vec);
  g.chunks = chunks_of(a.table, vec);
  const int rows = kThreads / g.lanes, all = a.Hq + a.Hk;
  const int64_t blocks = (static_cast<int64_t>(a.B) * a.T + rows - 1) / rows, once = static_cast<int64_t>(sms) * per_sm;
  // Heads are split until the blocks fill the GPU, down to one head.
  auto parts_of = [](int heads, int each) { return (heads + each - 1) / each; };
  int each = kHeadsEach;
  while (each > 1 && blocks * (parts_of(a.Hq, each) + parts_of(a.Hk, each)) < once) each /= 2;
  const int64_t full = blocks * (parts_of(a.Hq, each) + parts_of(a.Hk, each)) < kLong * once ? once : waves * once;
  auto set = [&](int heads, int& n, int& parts, int& share) {
    parts = parts_of(heads, each);
    share = parts_of(heads, parts);
    n = static_cast<int>(std::min(blocks, std::max<int64_t>(full * heads / all / parts, 1))) * parts;
  };
  set(a.Hq, g.q_blocks, g.q_parts, g.q_each);
  set(a.Hk, g.k_blocks, g.k_parts, g.k_each);
  return g;
}

template <int VEC, bool kBF16, int kLanes>
cudaError_t launch_fwd_t(const fa4d_norm_rotary_args& a, const NormGrid& g, cudaStream_t s) {
  auto kern = a.rotary.table.pairing == FA4D_PAIR_ADJACENT ? norm_rotary_kernel<kBF16, true, VEC, kLanes>
                                                           : norm_rotary_kernel<kBF16, false, VEC, kLanes>;
  constexpr int smem = Feed<VEC, true, 1, kFwdDepth>::kBytes;
  static_assert(smem <= 40 * 1024, "with what is static, more needs leave");
  return launch_chained(kern, dim3(g.q_blocks + g.k_blocks), kThreads, smem, 1, s, a, g);
}

template <int VEC, bool kBF16, int kLanes>
cudaError_t launch_bwd_t(const fa4d_norm_rotary_bwd_args& a, const NormGrid& g, cudaStream_t s) {
  auto kern = a.rotary.table.pairing == FA4D_PAIR_ADJACENT ? norm_rotary_grad_kernel<kBF16, true, VEC, kLanes>
                                                           : norm_rotary_grad_kernel<kBF16, false, VEC, kLanes>;
  constexpr int sums = kThreads * 2 * kRowPairs<VEC> * 4, feed = Feed<VEC, true, 2, kBwdDepth>::kBytes;
  constexpr int smem = feed > sums ? feed : sums;
  static_assert(smem <= 40 * 1024, "with what is static, more needs leave");
  const cudaError_t e =
      launch_chained(kern, dim3(g.q_blocks + g.k_blocks), kThreads, smem, 1, s, a, g);
  if (e != cudaSuccess) return e;
  const int D = a.rotary.table.D;
  return launch_chained(weight_grad_kernel<kBF16>, dim3((D + 7) / 8, 2), 256, 0, 1, s, static_cast<const float*>(a.workspace), D,
                        g.q_blocks, g.k_blocks, a.q_weight_grad, a.k_weight_grad, a.norm.weight_f32 != 0);
}

// The kernels of 4, 8 and 16 lanes a row (head dims from 33 to 256) know it, which saves the loops of
// their sums.
template <bool kBF16>
cudaError_t launch_fwd_b(const fa4d_norm_rotary_args& a, bool vec, int sms, cudaStream_t s) {
  const NormGrid g = grid_of(a.rotary, vec ? 8 : 1, kFwdPerSm, kFwdWaves, sms);
  if (!vec) return launch_fwd_t<1, kBF16, 32>(a, g, s);
  if (g.lanes == 16) return launch_fwd_t<8, kBF16, 16>(a, g, s);
  if (g.lanes == 8) return launch_fwd_t<8, kBF16, 8>(a, g, s);
  if (g.lanes == 4) return launch_fwd_t<8, kBF16, 4>(a, g, s);
  return launch_fwd_t<8, kBF16, 0>(a, g, s);
}
template <bool kBF16>
cudaError_t launch_bwd_b(const fa4d_norm_rotary_bwd_args& a, bool vec, int sms, cudaStream_t s) {
  const NormGrid g = grid_of(a.rotary, vec ? 8 : 1, kBwdPerSm, kBwdWaves, sms);
  if (!vec) return launch_bwd_t<1, kBF16, 32>(a, g, s);
  if (g.lanes == 16) return launch_bwd_t<8, kBF16, 16>(a, g, s);
  if (g.lanes == 8) return launch_bwd_t<8, kBF16, 8>(a, g, s);
  if (g.lanes == 4) return launch_bwd_t<8, kBF16, 4>(a, g, s);
  return launch_bwd_t<8, kBF16, 0>(a, g, s);
}

}  // namespace

// Rows of partial sums that a backward pass writes at most, whichever way its rows are divided: a
// block each (see grid_of: one a part where that is more than its share).
int64_t norm_bwd_rows(int Hq, int Hk, int sms) { return static_cast<int64_t>(sms) * kBwdPerSm * kBwdWaves + Hq + Hk; }

cudaError_t launch_norm_rotary(const fa4d_norm_rotary_args& a, bool vec, int sms, cudaStream_t s) {
  return a.rotary.dtype == FA4D_BF16 ? launch_fwd_b<true>(a, vec, sms, s) : launch_fwd_b<false>(a, vec, sms, s);
}

cudaError_t launch_norm_rotary_bwd(const fa4d_norm_rotary_bwd_args& a, bool vec, int sms, cudaStream_t s) {
  return a.rotary.dtype == FA4D_BF16 ? launch_bwd_b<true>(a, vec, sms, s) : launch_bwd_b<false>(a, vec, sms, s);
}

}  // namespace fa4d
