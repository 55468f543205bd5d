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
// them), then the requests' items (request, KV head, row tile), each with
// ceil(length / 16) units.  Warp w takes units [w q, (w + 1) q), so ragged lengths divide
// evenly without the host knowing them.  What warp w computes of an item is *segment*
// w + item (unique: along the line one of the two grows), an unnormalised fp32 output row
// with the running maximum (log2) and sum of its exponentials.
struct DecodeParams {
  const void* q;
  const void* pk;
  const void* pv;
  const void* k;
  const void* v;
  void* o;
  const int32_t* lengths;
  const uint8_t* mask;
  float* weights;
  int64_t q_stride[3], pk_stride[2], pv_stride[2], k_stride[3], v_stride[3], o_stride[3], mask_stride[3],
      weights_stride[2];
  int32_t B, T, Hq, Hk, P, C;
  int32_t G, R;
  int32_t tiles;         // row tiles of a (request, KV head)
  int32_t prefix_tiles;  // row tiles of a KV head's prefix in decode_kernel; 0: not done there
  int32_t prefix_units;  // units of a prefix item
  int32_t seg_rows;      // rows kept of a segment: min(16, R or the batch's rows)
  int32_t warps;         // warps of decode_kernel's grid
  int32_t min_units;     // least units of a warp
  int32_t causal;
  float scale_log2;      // scale * log2(e)
  float* seg_o;          // [segments][seg_rows][D]
  float2* seg_ml;        // [segments][seg_rows]: maximum (log2 units), sum
  float* logits;         // [B, Hk, R, logits_ld] of the own keys, log2 units; null without weights
  int32_t logits_ld;
  // Partial results of the prefix kernel: [Hk][splits][pre_rows] rows, splits 0: none.
  int32_t splits, pre_rows;
  float* pre_o;
  float2* pre_ml;
  int* status;
};

// Attention of all rows of each KV head over the prefix (fa4d_prefix.cu).
struct PrefixParams {
  CUtensorMap tm_k;  // dims (D, P, Hk, 1), box (64, 128, 1, 1), 128-B swizzle
  CUtensorMap tm_v;
  const void* q;
  int64_t q_stride[3];
  int32_t T, G, P, rows;  // rows of a KV head
  int32_t parts;          // partial results per row
  int32_t d_in;           // head dim of the tensors (96 computes at 128)
  float scale_log2;
  float* o;               // [Hk][parts][rows][d_in]
  float2* ml;             // [Hk][parts][rows]
  int* status;
};

constexpr int kDecodeWarps = 4;   // warps of a decode_kernel CTA
constexpr int kUnitKeys = 16;

cudaError_t launch_decode(const DecodeParams& p, int D, bool bf16, int ctas, bool after_prefix, cudaStream_t s);
// `split_keys`: the rows of a KV head fit one slot (at most 128), and a run's slots take even
// and odd key tiles; two parts per run then, one otherwise.
cudaError_t launch_prefix(const PrefixParams& p, int D, bool bf16, int Hk, int splits, bool split_keys, cudaStream_t s);
cudaError_t launch_join(const DecodeParams& p, int D, bool bf16, cudaStream_t s);
int decode_ctas_per_sm(int D);

}  // namespace fa4d
