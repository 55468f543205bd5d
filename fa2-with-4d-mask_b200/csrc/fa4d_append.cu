// fa4d_append.cu — the serving form of the norm with the rotary turn: new tokens join a cache of 16
// or 8 bits; and the values of an 8-bit cache in 16 bits.
#include <algorithm>

#include "fa4d.h"
#include "fa4d_cache8.cuh"
#include "fa4d_kernels.h"
#include "fa4d_launch.cuh"
#include "fa4d_norm.cuh"

namespace fa4d {

namespace {

constexpr int kRows = 16;  // rows of a block

// The blocks of a grid: first those of the caches, then q's.
struct AppendGrid {
  int chunks, lanes;
  uint32_t cache_blocks;
  uint32_t spans;      // 8-bit caches: 64-slot blocks that T tokens can touch
  uint32_t groups;     // of kRows tokens
  int q_each, k_each;  // heads of a block, of q and (16-bit caches) of k and of v
};

__device__ __forceinline__ int64_t entries_of(const fa4d_rotary_append_args& a, int64_t b) {
  return max(__ldcg(a.lengths + b), 0);
}
// The new length, and a cache that is full.
__device__ __forceinline__ void settle_length(const fa4d_rotary_append_args& a, int64_t b, int64_t had, int* status) {
  const int64_t now = had + a.T;
  a.lengths_out[b] = static_cast<int32_t>(min(now, static_cast<int64_t>(a.C)));
  if (now > a.C) atomicOr(status, FA4D_DEV_CACHE_FULL);
}

// q's rows: a group of tokens and a range of heads.
template <bool kBF16, bool kAdj, int VEC, int kHeads>
__device__ __forceinline__ void append_q(const fa4d_norm_append_args& args, const Turns<VEC>& turns, const Weights<VEC>& shared_w,
                                         const AppendGrid& g, uint32_t id) {
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1);
  const uint32_t n = static_cast<uint32_t>(id % g.groups) * kRows + threadIdx.x / g.lanes, T = a.T, b = n / T, t = n - b * T;
  const int first = id / g.groups * g.q_each;
  const bool live = n < a.B * T;
  const RowLane<VEC, kAdj> at(a.table, lane, g.chunks);
  const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1];
  uint16_t* dst = static_cast<uint16_t*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1];
  norm_heads<kBF16, kAdj, VEC, kHeads>(a.table, turns, at, args.norm.q_weight ? &shared_w : nullptr, args.norm.eps, g.lanes,
                                       lane, live, src, a.q_stride[2], dst, a.q_out_stride[2], first,
                                       min(first + g.q_each, a.Hq), a.positions, a.positions_bits, a.positions_stride, b, t);
}

// 16-bit caches.  A decode step has few tokens: everything is spread over the grid, and latency
// bounds it (160 tokens, Hq16 Hk4 D256: 4.0 us back to back; with four rows of q in flight, whose
// registers leave fewer blocks an SM, 4.5).  Two prompts of 4097 tokens (Hq32 Hk8 D128, 201 MB): 51.7 us,
// 59% of the measured copy rate; loads wait two heads at a time, with none fed ahead as in training.
template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 512) norm_append_kernel(const __grid_constant__ fa4d_norm_append_args args,
                                                                          const __grid_constant__ AppendGrid g, int* status) {
  __shared__ Turns<VEC> turns;
  turns.template fill<kAdj>(args.append.table);
  __syncthreads();
  pdl_wait();
  pdl_launch();
  __shared__ Weights<VEC> shared_w;
  uint32_t id = blockIdx.x;
  shared_w.template fill<kBF16, kAdj>(args.append.table, id >= g.cache_blocks ? args.norm.q_weight : args.norm.k_weight,
                                      args.norm.weight_f32 != 0);
  __syncthreads();
  if (id >= g.cache_blocks) return append_q<kBF16, kAdj, VEC, 2>(args, turns, shared_w, g, id - g.cache_blocks);
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1);
  const bool is_v = id >= g.cache_blocks / 2;
  id -= is_v ? g.cache_blocks / 2 : 0;
  const uint32_t n = static_cast<uint32_t>(id % g.groups) * kRows + threadIdx.x / g.lanes, T = a.T, b = n / T, t = n - b * T;
  const int first = id / g.groups * g.k_each, end = min(first + g.k_each, a.Hk);
  bool live = n < a.B * T;
  const int64_t had = live ? entries_of(a, b) : 0, slot = had + t;
  if (live && !is_v && first == 0 && t == 0 && lane == 0) settle_length(a, b, had, status);
  live = live && slot < a.C;
  const RowLane<VEC, kAdj> at(a.table, lane, g.chunks);
  if (is_v) {
    const uint16_t* src = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + t * a.v_stride[1];
    uint16_t* dst = static_cast<uint16_t*>(a.v_cache) + b * a.v_cache_stride[0] + slot * a.v_cache_stride[1];
    if (live)
      for (int h = first; h < end; ++h) {
        Raw<VEC> raw;
        at.load(src + h * a.v_stride[2], raw);
        at.store(dst + h * a.v_cache_stride[2], raw);
        if (a.weights && lane == 0) a.weights[b * a.weights_stride[0] + h * a.weights_stride[1] + slot] = 0.f;
      }
    return;
  }
  const uint16_t* src = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1];
  uint16_t* dst = static_cast<uint16_t*>(a.k_cache) + b * a.k_cache_stride[0] + slot * a.k_cache_stride[1];
  norm_heads<kBF16, kAdj, VEC, 2>(a.table, turns, at, &shared_w, args.norm.eps, g.lanes, lane, live, src, a.k_stride[2], dst,
                                  a.k_cache_stride[2], first, end, a.positions, a.positions_bits, a.positions_stride, b, t);
}

// 8-bit caches: a block of threads has a 64-slot block of one request, head and cache.  The new
// tokens' values wait in shared memory, in 32 bits, until their largest magnitude is known; then the
// scale, the earlier codes anew where it grows, and the new codes.  One token: latency, 3.1 us; 64
// tokens 6.9.  Two prompts of 4097 tokens (Hq32 Hk8 D128, 185 MB): 55.6 us, half of it q's rows.  Nothing
// is saturated there (issue slots 45%, DRAM 29%, 23% of the warps that an SM holds): 30 M warp
// instructions, the angles again for each KV head, and the waits of the two passes over their values (q by
// a kernel of its own, as in training: 2 us more).
template <bool kBF16, bool kAdj, int VEC, bool kInt8>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 512) append8_kernel(const __grid_constant__ fa4d_norm_append_args args,
                                                                      const __grid_constant__ AppendGrid g, int* status) {
  constexpr int P = kRowPairs<VEC>;
  extern __shared__ uint4 values[];  // [pass][P / 2][threads]: four values, two pairs
  __shared__ uint32_t block_most;
  __shared__ Turns<VEC> turns;
  uint32_t id = blockIdx.x;
  const bool is_v = id < g.cache_blocks && (id & 1);
  if (threadIdx.x == 0) block_most = 0;
  if (!is_v) turns.template fill<kAdj>(args.append.table);
  pdl_wait();
  pdl_launch();
  __shared__ Weights<VEC> shared_w;
  if (!is_v && args.norm.q_weight)
    shared_w.template fill<kBF16, kAdj>(args.append.table, id >= g.cache_blocks ? args.norm.q_weight : args.norm.k_weight,
                                        args.norm.weight_f32 != 0);
  __syncthreads();
  if (id >= g.cache_blocks) return append_q<kBF16, kAdj, VEC, 4>(args, turns, shared_w, g, id - g.cache_blocks);
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1), row = threadIdx.x / g.lanes, threads = blockDim.x;
  id >>= 1;
  const uint32_t row_of = id / g.spans, b = row_of / a.Hk;
  const int span = id - row_of * g.spans, h = row_of - b * a.Hk;
  const int64_t had = entries_of(a, b);
  if (h == 0 && span == 0 && !is_v && threadIdx.x == 0) settle_length(a, b, had, status);
  const int64_t block = had / FA4D_CACHE_BLOCK + span, start = block * FA4D_CACHE_BLOCK;
  const int64_t from = max(had, start), to = min(min(had + a.T, static_cast<int64_t>(a.C)), start + FA4D_CACHE_BLOCK);
  if (from >= to) return;

  const int64_t* ss = is_v ? args.v_scale_stride : args.k_scale_stride;
  float* scale_at = (is_v ? args.v_scale : args.k_scale) + b * ss[0] + h * ss[1] + block;
  const float old = from > start ? __ldcg(scale_at) : 0.f;
  const int64_t* st = is_v ? a.v_cache_stride : a.k_cache_stride;
  uint8_t* cache = static_cast<uint8_t*>(is_v ? a.v_cache : a.k_cache) + b * st[0] + h * st[2];
  const int64_t* xs = is_v ? a.v_stride : a.k_stride;
  const uint16_t* x = static_cast<const uint16_t*>(is_v ? a.v : a.k) + b * xs[0] + h * xs[2];
  const RowLane<VEC, kAdj> at(a.table, lane, g.chunks);
  const bool norm = !is_v && args.norm.k_weight;
  float largest = 0.f;
  const int count = static_cast<int>(to - from);
  Raw<VEC> raw;
  if (row < count) at.load(x + (from - had + row) * xs[1], raw);
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += kRows) {
    const bool live = i0 + row < count;
    const int64_t t = from - had + i0 + row;
    Pairs<VEC> p;
    unpack_pairs<kBF16, kAdj>(raw, p);
    if (i0 + kRows + row < count) at.load(x + (t + kRows) * xs[1], raw);  // on its way meanwhile
    // Keys with what roundings leave out, so that few of them come to lie on the wrong side of the border
    // of two codes.  Two prompts of 4097 tokens: of 8.4 million e4m3 keys 12.8 did without, 9.6 do
    // (means of 20 draws), for 55.6 us against 54.4; shorter appends take as long as without.
    Pairs<VEC> low;
#pragma unroll
    for (int j = 0; j < P / 2; ++j) low.a[j] = low.b[j] = f2(0.f, 0.f);
    if (norm) {
      const float square = row_sum(p.squares(), g.lanes);
      Pairs<VEC> w;
      at.weights(shared_w, lane, w);
      p.normalise(square * (1.f / a.table.D) + args.norm.eps, w, low);
    }
    if (!live) continue;
    if (!is_v) {
      Turn<VEC> turn;
      at.angles(turns, a.positions, a.positions_bits, a.positions_stride, b, t, lane, turn);
      turn.on_exact(p, low, at.copied());
    }
    uint4* v = values + i0 / kRows * (P / 2) * threads + threadIdx.x;
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      const float2 x0 = f2_split(p.a[j]), x1 = f2_split(p.b[j]);  // chunks past the last are zeros
      largest = max_abs_nan(max_abs_nan(largest, x0.x, x0.y), x1.x, x1.y);
      v[j * threads] = make_uint4(__float_as_uint(x0.x), __float_as_uint(x0.y), __float_as_uint(x1.x), __float_as_uint(x1.y));
    }
  }
  uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));  // NaN is above infinity
  if ((threadIdx.x & 31) == 0 && most) atomicMax(&block_most, most);
  __syncthreads();
  most = block_most;
  // The larger of the two, or NaN where either is (a block stays so while its earlier entries stay).
  float scale = least_scale<kInt8>(most);
  if (from > start && (old != old || scale <= old)) scale = old;
  if (threadIdx.x == 0 && (from == start || scale != old)) *scale_at = scale;
  if (from > start && scale > old) {  // codes of the earlier entries, 16 at a time
    const float factor = old / scale;
    const int parts = a.table.D / 16, all = static_cast<int>(from - start) * parts;
#pragma unroll 1
    for (int i = threadIdx.x; i < all; i += threads) {
      const int r = i / parts;
      uint4* at16 = reinterpret_cast<uint4*>(cache + (start + r) * st[1]) + (i - r * parts);
      uint4 c = __ldcg(at16);  // (a sector may hold another head's codes too, written by another SM)
      uint32_t* words = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[4];
        codes_to_float<kInt8>(words[k], f);
        words[k] = to_codes<kInt8>(f[0] * factor, f[1] * factor, f[2] * factor, f[3] * factor);
      }
      *at16 = c;
    }
  }
  const bool number = scale == scale;  // codes under a scale that is not are 0
  const float inverse = number ? 1.f / scale : 0.f;
  const uint64_t inverse2 = f2(inverse, inverse);
#pragma unroll 1
  for (int i0 = 0; i0 + row < count; i0 += kRows) {
    const uint4* v = values + i0 / kRows * (P / 2) * threads + threadIdx.x;
    uint8_t* dst = cache + (from + i0 + row) * st[1];
    float u[P], z[P];
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (number) x = v[j * threads];
      const float2 a2 = f2_split(fmul2(f2(__uint_as_float(x.x), __uint_as_float(x.y)), inverse2));
      const float2 b2 = f2_split(fmul2(f2(__uint_as_float(x.z), __uint_as_float(x.w)), inverse2));
      u[2 * j] = a2.x, u[2 * j + 1] = a2.y;
      z[2 * j] = b2.x, z[2 * j + 1] = b2.y;
    }
    if constexpr (VEC == 8) {
      if (!at.live) continue;
      uint2 lo, hi;
      if (kAdj) {
        lo = make_uint2(to_codes<kInt8>(u[0], z[0], u[1], z[1]), to_codes<kInt8>(u[2], z[2], u[3], z[3]));
        hi = make_uint2(to_codes<kInt8>(u[4], z[4], u[5], z[5]), to_codes<kInt8>(u[6], z[6], u[7], z[7]));
      } else {
        lo = make_uint2(to_codes<kInt8>(u[0], u[1], u[2], u[3]), to_codes<kInt8>(u[4], u[5], u[6], u[7]));
        hi = make_uint2(to_codes<kInt8>(z[0], z[1], z[2], z[3]), to_codes<kInt8>(z[4], z[5], z[6], z[7]));
      }
      *reinterpret_cast<uint2*>(dst + at.at0[0]) = lo;
      *reinterpret_cast<uint2*>(dst + at.at1[0]) = hi;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((at.live >> i) & 1u) {
          dst[at.at0[i]] = static_cast<uint8_t>(to_code<kInt8>(u[i]));
          dst[at.at1[i]] = static_cast<uint8_t>(to_code<kInt8>(z[i]));
        }
    }
  }
}

// n / d for n below 2^31 and d from 1: n * mul / 2^(32 + shift), with mul = ceil(2^(32 + shift) / d),
// 2^shift >= d / 2 (then mul < 2^32, and what it is too large by, times n, stays below 2^(32 + shift) / d).
struct Divisor {
  uint32_t mul, shift, d;
  explicit Divisor(uint32_t by) : mul(0), shift(0), d(by) {
    if (d == 1) return;
    while ((2u << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << (32 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

// One thread: kPieces times 8 codes, a block's threads apart, whose loads are in flight together.  1
// byte read and 2 written an element; two waits, for the length and for the codes, are a good part of
// a call's time (64 caches of 300 slots, Hk8 D128, half full: 12.9 us for 10 + 39 MB; 16 bytes a
// thread, one piece, 17 us; three to seven pieces differ by 8%).
constexpr int kPieces = 4, kValuesThreads = 128;
template <bool kBF16, bool kInt8>
__global__ void __launch_bounds__(kValuesThreads) cache_values_kernel(const __grid_constant__ fa4d_cache_values_args a, Divisor parts,
                                                           Divisor inner, bool heads_inner, uint32_t pieces) {
  pdl_wait();
  pdl_launch();
  const int64_t b = blockIdx.y;
  const int64_t length = __ldcg(a.lengths + b);
  const uint8_t* codes = static_cast<const uint8_t*>(a.codes) + b * a.codes_stride[0];
  const float* scales = a.scale + b * a.scale_stride[0];
  uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_stride[0];
  const uint32_t first = blockIdx.x * (kValuesThreads * kPieces) + threadIdx.x;
  uint2 c[kPieces];
  float scale[kPieces];
  int64_t to[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const uint32_t id = first + kValuesThreads * k, row = parts.of(id), part = id - row * parts.d;
    const uint32_t o = inner.of(row), i = row - o * inner.d;
    const int64_t slot = heads_inner ? o : i, h = heads_inner ? i : o;
    c[k] = make_uint2(0, 0);
    scale[k] = 0.f;
    if (id >= pieces) continue;
    to[k] = slot * a.out_stride[1] + h * a.out_stride[2] + 8 * part;
    if (slot >= length) continue;
    c[k] = __ldcg(reinterpret_cast<const uint2*>(codes + slot * a.codes_stride[1] + h * a.codes_stride[2]) + part);
    scale[k] = __ldcg(scales + h * a.scale_stride[1] + slot / FA4D_CACHE_BLOCK);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    if (first + kValuesThreads * k >= pieces) continue;
    float f[4], g[4];
    codes_to_float<kInt8>(c[k].x, f);
    codes_to_float<kInt8>(c[k].y, g);
    uint4 v;
    const uint64_t by = f2(scale[k], scale[k]);
    auto two = [&](float x, float y) {
      const float2 r = f2_split(fmul2(f2(x, y), by));
      return pack2<kBF16>(r.x, r.y);
    };
    v = make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(g[0], g[1]), two(g[2], g[3]));
    *reinterpret_cast<uint4*>(out + to[k]) = v;
  }
}

template <int VEC, bool kBF16, bool kAdj>
cudaError_t launch_append_t(const fa4d_norm_append_args& args, int sms, int* status, cudaStream_t s) {
  const fa4d_rotary_append_args& a = args.append;
  AppendGrid g;
  g.chunks = chunks_of(a.table, VEC);
  g.lanes = std::max(row_lanes(a.table, VEC), 2);  // whole warps
  const int threads = kRows * g.lanes;
  const int64_t tokens = static_cast<int64_t>(a.B) * a.T;
  g.groups = static_cast<uint32_t>((tokens + kRows - 1) / kRows);
  // One head a block until the blocks fill the GPU, then up to 16, which share the angles.
  auto each = [&](int heads) {
    int e = 1;
    while (e < 16 && static_cast<int64_t>(g.groups) * heads / (2 * e) >= 4LL * sms) e *= 2;
    return e;
  };
  g.q_each = each(a.Hq);
  g.k_each = each(a.Hk);
  const int64_t q_blocks = static_cast<int64_t>(g.groups) * ((a.Hq + g.q_each - 1) / g.q_each);
  int64_t cache_blocks;
  if (args.cache_type == FA4D_CACHE_16BIT) {
    g.spans = 0;
    cache_blocks = 2LL * g.groups * ((a.Hk + g.k_each - 1) / g.k_each);
  } else {
    g.spans = (a.T + FA4D_CACHE_BLOCK - 2) / FA4D_CACHE_BLOCK + 1;
    cache_blocks = 2LL * a.B * a.Hk * g.spans;
  }
  if (cache_blocks + q_blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  g.cache_blocks = static_cast<uint32_t>(cache_blocks);
  const dim3 grid(static_cast<unsigned>(cache_blocks + q_blocks));
  if (args.cache_type == FA4D_CACHE_16BIT)
    return launch_chained(norm_append_kernel<kBF16, kAdj, VEC>, grid, threads, 0, 1, s, args, g, status);
  const int passes = std::min((a.T + kRows - 1) / kRows, FA4D_CACHE_BLOCK / kRows);
  const size_t smem = static_cast<size_t>(passes) * (kRowPairs<VEC> / 2) * threads * sizeof(uint4);
  auto kern = args.cache_type == FA4D_CACHE_INT8 ? append8_kernel<kBF16, kAdj, VEC, true> : append8_kernel<kBF16, kAdj, VEC, false>;
  if (smem > 32 * 1024) {  // with what is static, 48 KB need no leave
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kern, grid, threads, smem, 1, s, args, g, status);
}

}  // namespace

cudaError_t launch_norm_append(const fa4d_norm_append_args& a, bool vec, int sms, int* status, cudaStream_t s) {
  const bool bf16 = a.append.dtype == FA4D_BF16, adj = a.append.table.pairing == FA4D_PAIR_ADJACENT;
  if (vec) {
    if (bf16) return adj ? launch_append_t<8, true, true>(a, sms, status, s) : launch_append_t<8, true, false>(a, sms, status, s);
    return adj ? launch_append_t<8, false, true>(a, sms, status, s) : launch_append_t<8, false, false>(a, sms, status, s);
  }
  if (bf16) return adj ? launch_append_t<1, true, true>(a, sms, status, s) : launch_append_t<1, true, false>(a, sms, status, s);
  return adj ? launch_append_t<1, false, true>(a, sms, status, s) : launch_append_t<1, false, false>(a, sms, status, s);
}

cudaError_t launch_cache_values(const fa4d_cache_values_args& a, cudaStream_t s) {
  // In the order of out's memory: heads within a slot where their stride is the smaller one.
  const bool heads_inner = a.out_stride[2] < a.out_stride[1];
  const Divisor parts(a.D / 8), inner(heads_inner ? a.Hk : a.C);
  const uint32_t pieces = static_cast<uint32_t>(static_cast<int64_t>(a.C) * a.Hk * (a.D / 8));  // fewer than 2^31 - 1024
  const dim3 grid((pieces + kValuesThreads * kPieces - 1) / (kValuesThreads * kPieces), a.B);
  const bool bf16 = a.dtype == FA4D_BF16, i8 = a.cache_type == FA4D_CACHE_INT8;
  auto kern = bf16 ? (i8 ? cache_values_kernel<true, true> : cache_values_kernel<true, false>)
                   : (i8 ? cache_values_kernel<false, true> : cache_values_kernel<false, false>);
  return launch_chained(kern, grid, kValuesThreads, 0, 1, s, a, parts, inner, heads_inner, pieces);
}

}  // namespace fa4d
