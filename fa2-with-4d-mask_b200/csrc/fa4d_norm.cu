// fa4d_norm.cu — training form of the norm of each head with the rotary turn in the same pass, and
// its gradient.
//
// Of a head x[D] with weights w: r = (mean x^2 + eps)^-1/2, y = turn(x r w).  Of dy, with
// g = turn^-1(dy):  dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x)).
// The backward pass works r out again from x, which it reads in any case.
//
// Bound by memory: the forward reads and writes each element once, the backward reads x and dy and
// writes dx.
#include "fa4d.h"
#include "fa4d_kernels.h"
#include "fa4d_launch.cuh"
#include "fa4d_norm.cuh"

namespace fa4d {

namespace {

constexpr int kThreads = 128;

// A block's part of the heads: q's first `q_parts` blocks along y, then k's.
struct HeadRange {
  bool is_q;
  int first, end;
  __device__ __forceinline__ HeadRange(int part, int q_parts, int each, int Hq, int Hk) {
    is_q = part < q_parts;
    first = (is_q ? part : part - q_parts) * each;
    end = min(first + each, is_q ? Hq : Hk);
  }
};

// One thread: a lane of a token's rows, for a range of q's or of k's heads, so that angles and
// weights serve several heads.
constexpr int kHeads = 4;

template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(kThreads) norm_rotary_kernel(const __grid_constant__ fa4d_norm_rotary_args args, int chunks,
                                                               int lanes, int q_parts, int heads_each) {
  const fa4d_rotary_args& a = args.rotary;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kThreads / lanes) + threadIdx.x / lanes;
  const bool live = n < static_cast<int64_t>(a.B) * a.T;
  const int64_t b = n / a.T, t = n - b * a.T;
  const HeadRange heads(blockIdx.y, q_parts, heads_each, a.Hq, a.Hk);
  const RowLane<VEC, kAdj> at(a.table, lane, chunks);
  pdl_wait();
  pdl_launch();
  Pairs<VEC> w;
  at.template vector<kBF16>(heads.is_q ? args.norm.q_weight : args.norm.k_weight, args.norm.weight_f32 != 0, w);
  const int64_t* si = heads.is_q ? a.q_stride : a.k_stride;
  const int64_t* so = heads.is_q ? a.q_out_stride : a.k_out_stride;
  const uint16_t* src = static_cast<const uint16_t*>(heads.is_q ? a.q : a.k) + b * si[0] + t * si[1];
  uint16_t* dst = static_cast<uint16_t*>(heads.is_q ? a.q_out : a.k_out) + b * so[0] + t * so[1];
  norm_heads<kBF16, kAdj, VEC, kHeads>(a.table, at, &w, args.norm.eps, lanes, lane, live, src, si[2], dst, so[2], heads.first,
                                       heads.end, a.positions, a.positions_bits, a.positions_stride, b, t);
}

// The gradient.  A block takes tokens gridDim.x * (rows of a block) apart and adds the weights'
// gradient up over all of them in registers, then over its rows in shared memory: one row of D sums
// a block, which weight_grad_kernel adds (always in the same order).
constexpr int kBwdHeads = 2;

template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(kThreads) norm_rotary_grad_kernel(const __grid_constant__ fa4d_norm_rotary_bwd_args args,
                                                                   int chunks, int lanes, int q_parts, int heads_each) {
  constexpr int P = kRowPairs<VEC>;
  __shared__ float sums[kThreads * 2 * P];  // [rows][D]
  const fa4d_rotary_args& a = args.rotary;
  const int lane = threadIdx.x & (lanes - 1), row = threadIdx.x / lanes, rows = kThreads / lanes;
  const HeadRange heads(blockIdx.y, q_parts, heads_each, a.Hq, a.Hk);
  const RowLane<VEC, kAdj> at(a.table, lane, chunks);
  pdl_wait();
  pdl_launch();
  Pairs<VEC> w, dw;
  at.template vector<kBF16>(heads.is_q ? args.norm.q_weight : args.norm.k_weight, args.norm.weight_f32 != 0, w);
#pragma unroll
  for (int j = 0; j < P; ++j) dw.a[j] = dw.b[j] = 0.f;
  const int64_t* si = heads.is_q ? a.q_stride : a.k_stride;
  const int64_t* sd = heads.is_q ? args.dq_stride : args.dk_stride;
  const int64_t* so = heads.is_q ? a.q_out_stride : a.k_out_stride;
  const uint16_t* x_all = static_cast<const uint16_t*>(heads.is_q ? a.q : a.k);
  const uint16_t* dy_all = static_cast<const uint16_t*>(heads.is_q ? args.dq : args.dk);
  uint16_t* dx_all = static_cast<uint16_t*>(heads.is_q ? a.q_out : a.k_out);
  const float mean = 1.f / a.table.D;
  const int64_t tokens = static_cast<int64_t>(a.B) * a.T;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.x) * rows; n0 < tokens; n0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t n = n0 + row;
    const bool live = n < tokens;
    const int64_t b = n / a.T, t = n - b * a.T;
    const uint16_t* x = x_all + b * si[0] + t * si[1];
    const uint16_t* dy = dy_all + b * sd[0] + t * sd[1];
    uint16_t* dx = dx_all + b * so[0] + t * so[1];
    float cs[P], sn[P];
    for (int h0 = heads.first; h0 < heads.end; h0 += kBwdHeads) {
      Raw<VEC> rx[kBwdHeads], rd[kBwdHeads];
#pragma unroll
      for (int u = 0; u < kBwdHeads; ++u)
        if (live && h0 + u < heads.end) {
          at.load(x + (h0 + u) * si[2], rx[u]);
          at.load(dy + (h0 + u) * sd[2], rd[u]);
        }
      if (h0 == heads.first && live) at.angles(a.table, a.positions, a.positions_bits, a.positions_stride, b, t, lane, cs, sn);
#pragma unroll
      for (int u = 0; u < kBwdHeads; ++u) {
        const bool here = live && h0 + u < heads.end;
        Pairs<VEC> xv, g;
        unpack_pairs<kBF16, kAdj>(rx[u], xv);
        unpack_pairs<kBF16, kAdj>(rd[u], g);
        if (here) at.turn(g, cs, sn, -1.f);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < P; ++j) dot = fmaf(xv.a[j], w.a[j] * g.a[j], fmaf(xv.b[j], w.b[j] * g.b[j], dot));
        float square = xv.squares();
        for (int o = lanes / 2; o; o >>= 1) {
          square += __shfl_xor_sync(0xffffffffu, square, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        if (!here) continue;
        const float r = rsqrtf(square * mean + args.norm.eps), c = r * r * (dot * mean);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          dw.a[j] = fmaf(g.a[j], xv.a[j] * r, dw.a[j]);
          dw.b[j] = fmaf(g.b[j], xv.b[j] * r, dw.b[j]);
          g.a[j] = r * (w.a[j] * g.a[j] - xv.a[j] * c);
          g.b[j] = r * (w.b[j] * g.b[j] - xv.b[j] * c);
        }
        pack_pairs<kBF16, kAdj>(g, rx[u]);
        at.store(dx + (h0 + u) * so[2], rx[u]);
      }
    }
  }
  // Over the block's rows.
#pragma unroll
  for (int i = 0; i < kRowChunks<VEC>; ++i)
    if ((at.live >> i) & 1u) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e0 = kAdj && VEC == 8 ? at.at0[i] + 2 * j : at.at0[i] + j, e1 = kAdj && VEC == 8 ? e0 + 1 : at.at1[i] + j;
        sums[row * a.table.D + e0] = dw.a[VEC * i + j];
        sums[row * a.table.D + e1] = dw.b[VEC * i + j];
      }
    }
  __syncthreads();
  float* part = static_cast<float*>(args.workspace) + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * a.table.D;
  for (int e = threadIdx.x; e < a.table.D; e += kThreads) {
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += sums[r * a.table.D + e];
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

struct NormGrid {
  int lanes, q_parts, each;
  dim3 grid;
};

NormGrid grid_of(const fa4d_rotary_args& a, int vec, int per_sm, int most_each, bool all_tokens, int sms) {
  NormGrid g;
  g.lanes = row_lanes(a.table, vec);
  const int rows = kThreads / g.lanes;
  const int64_t blocks = (static_cast<int64_t>(a.B) * a.T + rows - 1) / rows;
  // Heads are split until the blocks fill the GPU, down to one head.
  const int64_t full = static_cast<int64_t>(sms) * per_sm;
  g.each = most_each;
  while (g.each > 1 && blocks * ((a.Hq + g.each - 1) / g.each + (a.Hk + g.each - 1) / g.each) < full) g.each /= 2;
  g.q_parts = (a.Hq + g.each - 1) / g.each;
  const int parts = g.q_parts + (a.Hk + g.each - 1) / g.each;
  const int64_t x = all_tokens ? blocks : min(blocks, max(full / parts, static_cast<int64_t>(1)));
  g.grid = dim3(static_cast<unsigned>(x), parts);
  return g;
}

constexpr int kFwdPerSm = 12, kFwdEach = 8;
constexpr int kBwdPerSm = 4, kBwdEach = 8;

template <int VEC, bool kBF16>
cudaError_t launch_fwd_t(const fa4d_norm_rotary_args& a, int sms, cudaStream_t s) {
  const NormGrid g = grid_of(a.rotary, VEC, kFwdPerSm, kFwdEach, true, sms);
  auto kern = a.rotary.table.pairing == FA4D_PAIR_ADJACENT ? norm_rotary_kernel<kBF16, true, VEC>
                                                           : norm_rotary_kernel<kBF16, false, VEC>;
  return launch_chained(kern, g.grid, kThreads, 0, 1, s, a, chunks_of(a.rotary.table, VEC), g.lanes, g.q_parts, g.each);
}

template <int VEC, bool kBF16>
cudaError_t launch_bwd_t(const fa4d_norm_rotary_bwd_args& a, int sms, cudaStream_t s) {
  const NormGrid g = grid_of(a.rotary, VEC, kBwdPerSm, kBwdEach, false, sms);
  auto kern = a.rotary.table.pairing == FA4D_PAIR_ADJACENT ? norm_rotary_grad_kernel<kBF16, true, VEC>
                                                           : norm_rotary_grad_kernel<kBF16, false, VEC>;
  const cudaError_t e =
      launch_chained(kern, g.grid, kThreads, 0, 1, s, a, chunks_of(a.rotary.table, VEC), g.lanes, g.q_parts, g.each);
  if (e != cudaSuccess) return e;
  const int D = a.rotary.table.D, q_rows = g.q_parts * static_cast<int>(g.grid.x);
  const int k_rows = static_cast<int>(g.grid.y - g.q_parts) * static_cast<int>(g.grid.x);
  return launch_chained(weight_grad_kernel<kBF16>, dim3((D + 7) / 8, 2), 256, 0, 1, s, static_cast<const float*>(a.workspace), D,
                        q_rows, k_rows, a.q_weight_grad, a.k_weight_grad, a.norm.weight_f32 != 0);
}

}  // namespace

// Rows of partial sums that a backward pass writes at most, whichever way its rows are divided.
int64_t norm_bwd_rows(int Hq, int Hk, int sms) {
  const int64_t parts = Hq + Hk;  // one head each
  return max(static_cast<int64_t>(sms) * kBwdPerSm, parts);
}

cudaError_t launch_norm_rotary(const fa4d_norm_rotary_args& a, bool vec, int sms, cudaStream_t s) {
  const bool bf16 = a.rotary.dtype == FA4D_BF16;
  if (vec) return bf16 ? launch_fwd_t<8, true>(a, sms, s) : launch_fwd_t<8, false>(a, sms, s);
  return bf16 ? launch_fwd_t<1, true>(a, sms, s) : launch_fwd_t<1, false>(a, sms, s);
}

cudaError_t launch_norm_rotary_bwd(const fa4d_norm_rotary_bwd_args& a, bool vec, int sms, cudaStream_t s) {
  const bool bf16 = a.rotary.dtype == FA4D_BF16;
  if (vec) return bf16 ? launch_bwd_t<8, true>(a, sms, s) : launch_bwd_t<8, false>(a, sms, s);
  return bf16 ? launch_bwd_t<1, true>(a, sms, s) : launch_bwd_t<1, false>(a, sms, s);
}

}  // namespace fa4d
