// fa4d_decode.h — the division of shared-prefix attention into units and partial results,
// shared by the kernels that write them and the one that joins them.
#pragma once

#include <cstdint>
#include <cuda.h>

namespace fa4d {

// Rows of a (request, KV head): r = t * G + g, t a new token and g a query head of the KV
// head's group; R = T * G.  Rows of the prefix of a KV head: (b * T + t) * G + g over the
// whole batch.  Row tiles hold 16 rows.
//
// decode_kernel works on *units* of 16 keys of an *item* (a row tile with its keys), laid in
// one line: first the prefix items (KV head, row tile; none when the prefix kernel does
// them), then the requests' items (request, KV head, row tile), each with ceil(length / 16)
// units and the time of kItemUnits (of the prefix: kPrefixItemUnits) more, which a change of
// rows costs (its output written, the next item's queries read).  Each warp takes a run of the
// line (Shares), so ragged lengths divide evenly without the host knowing them.  What warp w
// computes of an item is *segment*
// w + item (unique: along the line one of the two grows), an unnormalised fp32 output row with
// the running maximum (log2) and sum of its exponentials: maximum -inf and sum 0 where the row saw
// no key (its output row may then be missing), and as part_of_keys writes them where it did.
// The run of a warp: the first `early` warps have `each` units, the others `late` (0: none); and
// the parts of a row that the prefix kernel made.  16 bytes, read together.
struct alignas(16) Shares {
  int32_t early, each, late, parts;
};

// What the prefix kernel takes of the GPU (see choose_runs).
struct PrefixLoad {
  int32_t items;  // CTAs per run of key tiles; 0: there is no prefix kernel
  int32_t most;   // runs of its grid
  int32_t tiles;  // 128-key tiles of the prefix
  int32_t step;   // key tiles that a CTA takes side by side
  int32_t sms;
  int32_t row_tiles;  // of a (request, KV head)
};

struct DecodeParams {
  CUtensorMap tm_k, tm_v;    // dims (D, C, Hk, B), box (64, 16, 1, 1), 128-B swizzle
  CUtensorMap tm_pk, tm_pv;  // the prefix (D, P, Hk, 1), where decode_kernel does it
  const void* q;
  void* o;
  const int32_t* lengths;
  const uint8_t* mask;
  float* weights;
  int64_t q_stride[3], o_stride[3], mask_stride[3], weights_stride[2];
  int32_t B, T, Hq, Hk, P, C;
  int32_t G, R;
  int32_t tiles;         // row tiles of a (request, KV head)
  int32_t prefix_tiles;  // row tiles of a KV head's prefix in decode_kernel; 0: not done there
  int32_t prefix_units;  // units of a prefix item
  int32_t unit_shift;    // keys of a unit, as a power of two: kUnitShift, or as the 8-bit kernel takes them
  int32_t seg_rows;      // rows kept of a segment: min(16, R or the batch's rows)
  int32_t heads;         // KV heads that neighbouring warps take side by side (decode8_kernel: 1, 2 or 4; otherwise 1)
  int32_t head_shift;    // log2(heads)
  int32_t groups;        // Hk / heads
  int32_t warps;         // warps of the grid / heads: those that take runs of the line
  int32_t min_units;     // least units of a warp
  PrefixLoad load;
  Shares* shares;        // written by decode_kernel (parts: by prefix_kernel), read by the join
  int32_t causal;
  float scale_log2;      // scale * log2(e)
  float* seg_o;          // [segments][seg_rows][D]
  float2* seg_ml;        // [segments][seg_rows]: maximum (log2 units), sum
  float* logits;         // [B, Hk, R, logits_ld] of the own keys, log2 units; null without weights
  int32_t logits_ld;
  int32_t weights_vec;   // rows of weights start on 16-byte boundaries
  float* lse;            // [B, Hk, R]: log2 of a row's sum, written by the join with weights; +inf without a key
  // Partial results of the prefix kernel: [Hk][splits][pre_rows] rows, splits 0: none.
  int32_t splits, pre_rows;
  float* pre_o;
  float2* pre_ml;
  int* status;
};

// The same over caches in 8 bits (fa4d_decode8.cu): tm_k, tm_v over bytes, no weights, no prefix items.
struct Decode8Params {
  DecodeParams d;
  const float* k_scale;
  const float* v_scale;
  int64_t k_scale_stride[2], v_scale_stride[2];
  int32_t q_bf16;
};

// Attention of all rows of each KV head over the prefix (fa4d_prefix.cu).
struct PrefixParams {
  CUtensorMap tm_k;  // dims (D, P, Hk, 1), box (64, 128, 1, 1), 128-B swizzle
  CUtensorMap tm_v;
  const void* q;
  int64_t q_stride[3];
  int32_t T, G, P, rows;  // rows of a KV head
  int32_t parts;          // partial results per row, at most
  const int32_t* lengths;  // of the own keys that the decode kernel reads meanwhile
  int32_t B, C, Hk;
  int32_t unit_shift;
  PrefixLoad load;
  Shares* shares;         // `parts` written: the partial results per row, at most p.parts
  int32_t d_in;           // head dim of the tensors (96 computes at 128)
  float scale_log2;
  float* o;               // [Hk][parts][rows][d_in]
  float2* ml;             // [Hk][parts][rows]
  int* status;
};

constexpr int kDecodeWarps = 4;   // warps of a decode_kernel CTA
constexpr int kUnitShift = 4;     // keys of a unit of decode_kernel, as a power of two
constexpr int kUnitKeys = 1 << kUnitShift;
// Of decode8_kernel: K and V of 8 KB, as decode_kernel's at head dim 128.
template <int D>
constexpr int kUnit8Shift = D == 64 ? 6 : D == 256 ? 4 : 5;
// Its column tiles of 8 rows, and its CTAs of an SM: as many as the registers allow, since a unit is a
// chain of waits (about 1600 clocks) that only other warps fill (1.2 GB of codes, B64 Hk8 D128, 4 rows:
// 231 us with two CTAs and three stages a warp, 186 with three and two).
inline int decode8_cols(int64_t R) { return R <= 8 ? 1 : 2; }
template <int D, int kCols>
constexpr int kCtas8 = kCols == 1 && D <= 128 ? 3 : 2;
constexpr int kItemUnits = 2;
// The prefix's items lie together at the front: with a short prefix the first warps do little but
// change rows, each time with a wait as long as memory is busy (128 requests, 918 MB of own keys,
// 16 prefix keys: 226 us with 2, 198 with 6, 177 with 12, 165 with 20; small calls lose 1% from 6
// to 12 and again to 20).
constexpr int kPrefixItemUnits = 8;

// Measured on B200, in microseconds: a key tile of a prefix kernel CTA (two of them, taken side
// by side, where the slots split the keys) and a CTA's fill, drain and output rows; a unit of a
// decode_kernel warp beside the SM's others, and the time until its first unit.
template <int D>
constexpr float kTileMicros = D == 256 ? 1.75f : D == 64 ? 1.9f : 2.1f;
constexpr float kRunMicros = 6.0f;
template <int D>
constexpr float kUnitMicros = D == 256 ? 1.0f : D == 64 ? 0.8f : 1.1f;
constexpr float kDecodeMicros = 3.5f;
constexpr float kReadRate = 6.0f;  // MB per microsecond that decode_kernel reads, of the GPU
constexpr float kPrefixWeight = 0.1f;  // see choose_runs
template <int D>
constexpr int kDecodeCtas = D == 256 ? 1 : 2;  // of an SM

#ifdef __CUDACC__
// The maximum and sum of a part that saw keys.  A maximum leaves NaN out, so a sum over keys of
// logit NaN alone comes with the maximum -inf: it becomes 0, and the sum reaches every sum that it
// is joined to.  Keys of logit -inf alone sum to 0: the part counts for nothing beside a finite
// logit, but a row of such parts is undefined, which the sum 1 tells from a row without a key.
__device__ __forceinline__ void part_of_keys(float& m, float& l) {
  if (m != -INFINITY) return;
  if (l != l)
    m = 0.f;
  else
    l = 1.f;
}

struct RunChoice {
  int runs;
  float prefix_us, total_us;  // of the prefix kernel, of both
  float rate;                 // units per microsecond of the whole GPU
};

// Read past L1 (as is everything that a kernel of the chain reads without a wait of its own):
// what is complete is in L2, and an SM's L1 may still hold what an earlier kernel read there.
__device__ __forceinline__ int length_at(const int32_t* lengths, int b, int C) { return min(max(__ldcg(lengths + b), 0), C); }
// Units of 2^shift keys.
__device__ __forceinline__ int units_of(int keys, int shift) { return (keys + (1 << shift) - 1) >> shift; }

// What an item of so many keys takes of the line.
__device__ __forceinline__ int line_of(int keys, int shift) { return keys > 0 ? units_of(keys, shift) + kItemUnits : 0; }

// a / b for a >= 0, b > 0, in 32 bits where that does (a 64-bit division is five times as long).
__device__ __forceinline__ int64_t quotient(int64_t a, int b) {
  return a >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

// The division of `total` units among so many warps where no prefix kernel runs beside them.
__device__ __forceinline__ Shares even_shares(int64_t total, int warps, int least) {
  return Shares{warps, max(static_cast<int>(quotient(total + warps - 1, warps)), least), 0, 0};
}

// What the requests before b (all of them for b = B) take of the line, per KV head and row tile.
__device__ __forceinline__ int64_t line_before(const int32_t* lengths, int C, int b, int lane, int shift) {
  int64_t n = 0;
  for (int i = lane; i < b; i += 128) {  // four loads in flight
    int u[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) u[x] = line_of(length_at(lengths, min(i + 32 * x, b - 1), C), shift);
#pragma unroll
    for (int x = 0; x < 4; ++x) n += i + 32 * x < b ? u[x] : 0;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// How many runs the prefix's key tiles are divided into, at most the grid's.  A run fills an SM
// (shared memory and registers), and the decode kernel, launched right behind, streams the own
// keys (`units` of them) on the SMs that are left: fewer, longer runs let the tensor work and
// the memory work go on side by side.  Only the lengths, on the device, tell how much that is,
// so it is worked out there by one warp (lane l for l + 1, l + 33, ... runs).  Where the own
// keys take longer than the prefix whatever its runs, the estimates of many divisions are
// equal; what they leave out (the start of the CTAs that come late) goes with the prefix
// kernel's time, a part of which is therefore added; of equal divisions the one with fewer
// partial rows to join is taken.  Over 18 calls (8 to 256 requests, 1024 to 30000 prefix keys,
// head dims 64 to 256), each timed with every number of runs, the choice is 1.0% above the best
// on average and 4% at most (3.3% and 25% with the larger of equal numbers of runs and without
// that part).  Those calls had 16-bit caches.  Before own caches in 8 bits the choice is made with the same
// numbers, which are not fitted to decode8_kernel: a unit is 8 KB there for head dims 64, 128 and 256 (4,
// 8 and 16 KB here), takes 1.6 to 1.9 us of a warp, and an SM holds three CTAs up to 8 rows.  That costs
// time at most: both kernels divide by what is found here, whatever it is.
template <int D>
__device__ __forceinline__ RunChoice choose_runs(const PrefixLoad& w, int64_t units, int lane) {
  const float all = static_cast<float>(units);
  const float sm_rate = kDecodeCtas<D> * kDecodeWarps / kUnitMicros<D>;
  // Row tiles of a request read the same keys, mostly from L2.
  const float gpu_rate = fminf(w.sms * sm_rate, kReadRate * 1e6f / (kUnitKeys * 4 * D) * w.row_tiles);
  RunChoice best{1, 0.f, 0.f, gpu_rate};
  float best_cost = INFINITY;
  for (int s = lane + 1; s <= w.most; s += 32) {
    const int ctas = w.items * s, run = (w.tiles + s - 1) / s;
    const float mine = ((ctas + w.sms - 1) / w.sms) * (((run + w.step - 1) / w.step) * kTileMicros<D> + kRunMicros);
    const float beside = fminf(gpu_rate, sm_rate * max(w.sms - ctas, 0)) * fmaxf(mine - kDecodeMicros, 0.f);
    const float total = mine + (all > beside ? kDecodeMicros + (all - beside) / gpu_rate : 0.f);
    if (total + kPrefixWeight * mine < best_cost) {
      best_cost = total + kPrefixWeight * mine;
      best.runs = s;
      best.prefix_us = mine;
      best.total_us = total;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const int s = __shfl_xor_sync(0xffffffffu, best.runs, o);
    const float cost = __shfl_xor_sync(0xffffffffu, best_cost, o);
    const float mine = __shfl_xor_sync(0xffffffffu, best.prefix_us, o);
    const float total = __shfl_xor_sync(0xffffffffu, best.total_us, o);
    if (cost < best_cost || (cost == best_cost && s < best.runs)) {
      best_cost = cost;
      best.runs = s;
      best.prefix_us = mine;
      best.total_us = total;
    }
  }
  return best;
}
#endif

cudaError_t launch_decode(const DecodeParams& p, int D, bool bf16, int ctas, bool after_prefix, cudaStream_t s);
cudaError_t launch_decode8(const Decode8Params& p, int D, bool int8, int ctas, bool after_prefix, cudaStream_t s);
// `split_keys`: the rows of a KV head fit one slot (at most 128), and a run's slots take even
// and odd key tiles; two parts per run then, one otherwise.
cudaError_t launch_prefix(const PrefixParams& p, int D, bool bf16, int Hk, int splits, bool split_keys, cudaStream_t s);
cudaError_t launch_join(const DecodeParams& p, int D, bool bf16, int sms, cudaStream_t s);

}  // namespace fa4d
