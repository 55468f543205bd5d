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
  int cache_blocks;
  int spans;                // 8-bit caches: 64-slot blocks that T tokens can touch
  int groups;               // of kRows tokens
  int q_each, k_each;       // heads of a block, of q and (16-bit caches) of k and of v
  int q_parts, k_parts;
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
template <bool kBF16, bool kAdj, int VEC>
__device__ __forceinline__ void append_q(const fa4d_norm_append_args& args, const Turns<VEC>& turns, const Weights<VEC>& shared_w,
                                         const AppendGrid& g, int id) {
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1);
  const int64_t n = static_cast<int64_t>(id % g.groups) * kRows + threadIdx.x / g.lanes;
  const int first = id / g.groups * g.q_each;
  const bool live = n < static_cast<int64_t>(a.B) * a.T;
  const int64_t b = n / a.T, t = n - b * a.T;
  const RowLane<VEC, kAdj> at(a.table, lane, g.chunks);
  const uint16_t* src = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1];
  uint16_t* dst = static_cast<uint16_t*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1];
  norm_heads<kBF16, kAdj, VEC, 4>(a.table, turns, at, args.norm.q_weight ? &shared_w : nullptr, args.norm.eps, g.lanes, lane, live, src,
                                  a.q_stride[2], dst, a.q_out_stride[2], first, min(first + g.q_each, a.Hq), a.positions,
                                  a.positions_bits, a.positions_stride, b, t);
}

// 16-bit caches.  A decode step has few tokens: everything is spread over the grid, and latency
// bounds it.
template <bool kBF16, bool kAdj, int VEC>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 512) norm_append_kernel(const __grid_constant__ fa4d_norm_append_args args,
                                                                          const __grid_constant__ AppendGrid g, int* status) {
  __shared__ Turns<VEC> turns;
  turns.template fill<kAdj>(args.append.table);
  __syncthreads();
  pdl_wait();
  pdl_launch();
  __shared__ Weights<VEC> shared_w;
  int id = blockIdx.x;
  shared_w.template fill<kBF16, kAdj>(args.append.table, id >= g.cache_blocks ? args.norm.q_weight : args.norm.k_weight,
                                      args.norm.weight_f32 != 0);
  __syncthreads();
  if (id >= g.cache_blocks) return append_q<kBF16, kAdj, VEC>(args, turns, shared_w, g, id - g.cache_blocks);
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1);
  const bool is_v = id >= g.cache_blocks / 2;
  id -= is_v ? g.cache_blocks / 2 : 0;
  const int64_t n = static_cast<int64_t>(id % g.groups) * kRows + threadIdx.x / g.lanes;
  const int first = id / g.groups * g.k_each, end = min(first + g.k_each, a.Hk);
  bool live = n < static_cast<int64_t>(a.B) * a.T;
  const int64_t b = n / a.T, t = n - b * a.T;
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
  norm_heads<kBF16, kAdj, VEC, 4>(a.table, turns, at, &shared_w, args.norm.eps, g.lanes, lane, live, src, a.k_stride[2], dst,
                                  a.k_cache_stride[2], first, end, a.positions, a.positions_bits, a.positions_stride, b, t);
}

// 8-bit caches: a block of threads has a 64-slot block of one request, head and cache.  The new
// tokens' values wait in shared memory, in 32 bits, until their largest magnitude is known; then the
// scale, the earlier codes anew where it grows, and the new codes.
template <bool kBF16, bool kAdj, int VEC, bool kInt8>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 512) append8_kernel(const __grid_constant__ fa4d_norm_append_args args,
                                                                      const __grid_constant__ AppendGrid g, int* status) {
  constexpr int P = kRowPairs<VEC>;
  extern __shared__ float values[];  // [pass][2 P][threads]
  __shared__ uint32_t block_most;
  __shared__ Turns<VEC> turns;
  if (threadIdx.x == 0) block_most = 0;
  turns.template fill<kAdj>(args.append.table);
  __syncthreads();
  pdl_wait();
  pdl_launch();
  __shared__ Weights<VEC> shared_w;
  int64_t id = blockIdx.x;
  if (args.norm.q_weight)
    shared_w.template fill<kBF16, kAdj>(args.append.table, id >= g.cache_blocks ? args.norm.q_weight : args.norm.k_weight,
                                        args.norm.weight_f32 != 0);
  __syncthreads();
  if (id >= g.cache_blocks) return append_q<kBF16, kAdj, VEC>(args, turns, shared_w, g, static_cast<int>(id - g.cache_blocks));
  const fa4d_rotary_append_args& a = args.append;
  const int lane = threadIdx.x & (g.lanes - 1), row = threadIdx.x / g.lanes, threads = blockDim.x;
  const bool is_v = id & 1;
  id >>= 1;
  const int span = static_cast<int>(id % g.spans);
  id /= g.spans;
  const int h = static_cast<int>(id % a.Hk);
  const int64_t b = id / a.Hk;
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
  uint32_t most = 0;
  const int count = static_cast<int>(to - from);
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += kRows) {
    const bool live = i0 + row < count;
    const int64_t t = from - had + i0 + row;
    Raw<VEC> raw;
    if (live) at.load(x + t * xs[1], raw);
    Pairs<VEC> p;
    unpack_pairs<kBF16, kAdj>(raw, p);
    if (norm) p.times(rsqrtf(row_sum(p.squares(), g.lanes) * (1.f / a.table.D) + args.norm.eps));
    if (!live) continue;
    if (!is_v) {
      Turn<VEC> turn;
      at.angles(turns, a.positions, a.positions_bits, a.positions_stride, b, t, lane, turn);
      Pairs<VEC> w;
      if (norm) at.weights(shared_w, lane, w);
      Factors<VEC> factors;
      factors.set(turn, norm ? &w : nullptr);
      factors.turn(p, at.copied());
    }
    float* v = values + i0 / kRows * (2 * P) * threads + threadIdx.x;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      // Dead chunks hold zeros.
      const float2 u = f2_split(p.a[j / 2]), z = f2_split(p.b[j / 2]);
      const float x0 = j & 1 ? u.y : u.x, x1 = j & 1 ? z.y : z.x;
      most = max(most, max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu));
      v[j * threads] = x0;
      v[(P + j) * threads] = x1;
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
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
      uint4 c = *at16;
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
  const float inverse = 1.f / scale;
#pragma unroll 1
  for (int i0 = 0; i0 + row < count; i0 += kRows) {
    const float* v = values + i0 / kRows * (2 * P) * threads + threadIdx.x;
    uint8_t* dst = cache + (from + i0 + row) * st[1];
    float u[P], z[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      u[j] = number ? v[j * threads] * inverse : 0.f;
      z[j] = number ? v[(P + j) * threads] * inverse : 0.f;
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

// One thread: 16 codes of a slot and head.  Bound by memory: 1 byte read and 2 written an element.
template <bool kBF16, bool kInt8>
__global__ void __launch_bounds__(256) cache_values_kernel(const __grid_constant__ fa4d_cache_values_args a, int parts) {
  pdl_wait();
  pdl_launch();
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  const int64_t b = blockIdx.y;
  // In the order of out's memory: heads within a slot where their stride is the smaller one.
  const bool heads_inner = a.out_stride[2] < a.out_stride[1];
  const uint32_t row = id / parts, part = id - row * parts;
  const uint32_t inner = heads_inner ? a.Hk : a.C;
  const uint32_t o = row / inner, i = row - o * inner;
  if (o >= static_cast<uint32_t>(heads_inner ? a.C : a.Hk)) return;
  const int64_t slot = heads_inner ? o : i, h = heads_inner ? i : o;
  uint4 out[2] = {};
  if (slot < __ldcg(a.lengths + b)) {
    const uint4 c = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.codes) + b * a.codes_stride[0] +
                                                          slot * a.codes_stride[1] + h * a.codes_stride[2]) + part);
    const float scale = __ldcg(a.scale + b * a.scale_stride[0] + h * a.scale_stride[1] + slot / FA4D_CACHE_BLOCK);
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
    uint32_t* to = reinterpret_cast<uint32_t*>(out);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[4];
      codes_to_float<kInt8>(words[k], f);
      to[2 * k] = pack2<kBF16>(f[0] * scale, f[1] * scale);
      to[2 * k + 1] = pack2<kBF16>(f[2] * scale, f[3] * scale);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + b * a.out_stride[0] + slot * a.out_stride[1] +
                                        h * a.out_stride[2]) + 2 * part;
  dst[0] = out[0];
  dst[1] = out[1];
}

template <int VEC, bool kBF16, bool kAdj>
cudaError_t launch_append_t(const fa4d_norm_append_args& args, int sms, int* status, cudaStream_t s) {
  const fa4d_rotary_append_args& a = args.append;
  AppendGrid g;
  g.chunks = chunks_of(a.table, VEC);
  g.lanes = std::max(row_lanes(a.table, VEC), 2);  // whole warps
  const int threads = kRows * g.lanes;
  const int64_t tokens = static_cast<int64_t>(a.B) * a.T;
  g.groups = static_cast<int>((tokens + kRows - 1) / kRows);
  // One head a block until the blocks fill the GPU, then up to 8, which share the angles.
  auto each = [&](int heads) {
    int e = 1;
    while (e < 8 && static_cast<int64_t>(g.groups) * heads / (2 * e) >= 8LL * sms) e *= 2;
    return e;
  };
  g.q_each = each(a.Hq);
  g.k_each = each(a.Hk);
  g.q_parts = (a.Hq + g.q_each - 1) / g.q_each;
  g.k_parts = (a.Hk + g.k_each - 1) / g.k_each;
  const int64_t q_blocks = static_cast<int64_t>(g.groups) * g.q_parts;
  int64_t cache_blocks;
  if (args.cache_type == FA4D_CACHE_16BIT) {
    g.spans = 0;
    cache_blocks = 2LL * g.groups * g.k_parts;
  } else {
    g.spans = (a.T + FA4D_CACHE_BLOCK - 2) / FA4D_CACHE_BLOCK + 1;
    cache_blocks = 2LL * a.B * a.Hk * g.spans;
  }
  if (cache_blocks + q_blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  g.cache_blocks = static_cast<int>(cache_blocks);
  const dim3 grid(static_cast<unsigned>(cache_blocks + q_blocks));
  if (args.cache_type == FA4D_CACHE_16BIT)
    return launch_chained(norm_append_kernel<kBF16, kAdj, VEC>, grid, threads, 0, 1, s, args, g, status);
  const int passes = std::min((a.T + kRows - 1) / kRows, FA4D_CACHE_BLOCK / kRows);
  const size_t smem = static_cast<size_t>(passes) * 2 * kRowPairs<VEC> * threads * sizeof(float);
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
  const int parts = a.D / 16;
  const int64_t threads = static_cast<int64_t>(a.C) * a.Hk * parts;  // fewer than 2^31, B at most 65535
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256), a.B);
  const bool bf16 = a.dtype == FA4D_BF16, i8 = a.cache_type == FA4D_CACHE_INT8;
  auto kern = bf16 ? (i8 ? cache_values_kernel<true, true> : cache_values_kernel<true, false>)
                   : (i8 ? cache_values_kernel<false, true> : cache_values_kernel<false, false>);
  return launch_chained(kern, grid, 256, 0, 1, s, a, parts);
}

}  // namespace fa4d
