// fa4d_cache_api.cu — the C ABI of the operators around the attention: rotary positions and
// their serving form, attention over a shared prefix and own caches, eviction.  Argument
// checks, the division of work and dispatch; nothing is allocated here.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "fa4d.h"
#include "fa4d_decode.h"
#include "fa4d_host.h"
#include "fa4d_kernels.h"

namespace {

using fa4d::host_bind_device_of;
using fa4d::host_ok;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return fa4d::host_fail(code, buf);
}

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return fail(FA4D_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  return host_ok();
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Rows of a 16-bit tensor that 16-byte accesses can reach.
bool rows16(const void* p, const int64_t* st, int n) {
  bool ok = aligned16(p);
  for (int i = 0; i < n; ++i) ok = ok && st[i] % 8 == 0;
  return ok;
}

int check_dtype(int dtype) {
  if (dtype != FA4D_BF16 && dtype != FA4D_F16) return fail(FA4D_ERR_INVALID, "dtype %d is not bf16/f16", dtype);
  return FA4D_OK;
}

int check_table(const fa4d_rotary_table& t, int positions_bits) {
  if (t.D < 2 || t.D % 2 || t.D > 2 * FA4D_ROTARY_MAX_PAIRS)
    return fail(FA4D_ERR_UNSUPPORTED, "head dim %d must be even and at most %d", t.D, 2 * FA4D_ROTARY_MAX_PAIRS);
  if (t.rotary_dim < 2 || t.rotary_dim % 2 || t.rotary_dim > t.D)
    return fail(FA4D_ERR_INVALID, "rotary_dim %d must be even and in [2, %d]", t.rotary_dim, t.D);
  if (t.pairing != FA4D_PAIR_HALF && t.pairing != FA4D_PAIR_ADJACENT)
    return fail(FA4D_ERR_INVALID, "pairing %d is unknown", t.pairing);
  for (int i = 0; i < t.rotary_dim / 2; ++i)
    if (t.axis[i] >= t.axes) return fail(FA4D_ERR_INVALID, "pair %d has axis %d of %d", i, t.axis[i], t.axes);
  if (positions_bits != 32 && positions_bits != 64)
    return fail(FA4D_ERR_INVALID, "positions_bits %d is not 32 or 64", positions_bits);
  return FA4D_OK;
}

// Runs of 8 pairs, and of 16 copied elements.
bool table_vec(const fa4d_rotary_table& t) { return t.rotary_dim % 16 == 0 && t.D % 16 == 0; }

// Everything the prefix attention derives from the sizes.
struct Plan {
  fa4d::DecodeParams p;
  int ctas;
  int splits;        // runs of key tiles of the prefix kernel; 0: decode_kernel does the prefix
  bool split_keys;
  size_t seg_o, seg_ml, logits, lse, pre_o, pre_ml, shares, total;
};

// Runs per (row tile, KV head) of the prefix kernel: the number that shortens the estimate
// waves x (tiles of a run x time of a tile + fixed time of a CTA) + the partial rows written
// and read back.
int prefix_splits(int64_t row_tiles, int Hk, int tiles, int64_t rows, int D, bool split_keys, int sms) {
  // Microseconds: a key tile of a CTA (two at a time with split_keys), and its fill, drain and
  // output rows; measured on B200.
  const double fixed = fa4d::kRunMicros;
  const double tile = D == 256 ? fa4d::kTileMicros<256> : D == 64 ? fa4d::kTileMicros<64> : fa4d::kTileMicros<128>;
  const int step = split_keys ? 2 : 1;
  double best = 0.0;
  int best_s = 1;
  for (int s = 1; s <= tiles && s <= 64; ++s) {
    const double waves = std::ceil(static_cast<double>(row_tiles) * Hk * s / sms);
    const int run = (tiles + s - 1) / s;
    const double t = waves * ((run + step - 1) / step * tile + fixed) + 1.6e-6 * step * s * rows * Hk * D;
    if (s == 1 || t < best) {
      best = t;
      best_s = s;
    }
  }
  return best_s;
}

// decode_kernel reads the prefix once per 16 rows, from L2 after the first time, and spares the
// prefix kernel's launch and start.  It takes the prefix while what it reads of K (V as much
// again) is at most this many elements.  Both ways (here / prefix kernel), in us, behind own
// caches of 100, Hq32 Hk8 D128: 16 rows 14.0 / 15.2 at P 2048 and 23.2 / 19.8 at 8192; 64 rows
// 15.5 / 15.5 at 512 and 19.0 / 17.3 at 2048; Hq64 Hk1 D64, 128 rows: 11.0 / 14.2 at 2048 and
// 24.7 / 18.9 at 32768; Hq16 Hk4 D256, 128 rows: 16.9 / 18.1 at 512 and 24.5 / 21.8 at 2048.
constexpr int64_t kDecodePrefix = 1 << 22;

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

int plan_prefix(int B, int T, int Hq, int Hk, int D, int P, int C, bool weights, Plan* out) {
  if (B < 1 || T < 1 || Hq < 1 || Hk < 1 || C < 1 || P < 0)
    return fail(FA4D_ERR_INVALID, "sizes must be positive (B=%d T=%d Hq=%d Hk=%d C=%d P=%d)", B, T, Hq, Hk, C, P);
  if (Hq % Hk != 0) return fail(FA4D_ERR_INVALID, "query heads (%d) must be divisible by key/value heads (%d)", Hq, Hk);
  if (D != 64 && D != 96 && D != 128 && D != 256)
    return fail(FA4D_ERR_UNSUPPORTED, "head dim %d is not built (64, 96, 128, 256)", D);
  if (B > 65535 || Hk > 65535) return fail(FA4D_ERR_UNSUPPORTED, "B and Hk must be <= 65535");
  if (P > (1 << 30) || C > (1 << 30)) return fail(FA4D_ERR_UNSUPPORTED, "more than 2^30 keys");
  const int64_t rows = static_cast<int64_t>(B) * T * (Hq / Hk);
  if (rows > (1 << 26)) return fail(FA4D_ERR_UNSUPPORTED, "more than 2^26 query rows of a key/value head");
  memset(out, 0, sizeof(*out));
  fa4d::DecodeParams& p = out->p;
  p.B = B, p.T = T, p.Hq = Hq, p.Hk = Hk, p.P = P, p.C = C;
  p.G = Hq / Hk;
  p.R = T * p.G;
  p.tiles = (p.R + 15) / 16;
  const int sms = fa4d::host_sm_count();
  if ((rows + 15) / 16 * P * Hk * D > kDecodePrefix) {
    out->split_keys = D != 256 && rows <= 128;
    const int64_t row_tiles = D == 256 || out->split_keys ? (rows + 127) / 128 : (rows + 255) / 256;
    out->splits = prefix_splits(row_tiles, Hk, (P + 127) / 128, rows, D, out->split_keys, sms);
    p.splits = out->splits * (out->split_keys ? 2 : 1);
    p.pre_rows = static_cast<int>(rows);
    p.load = fa4d::PrefixLoad{static_cast<int>(row_tiles) * Hk, out->splits, (P + 127) / 128, out->split_keys ? 2 : 1, sms,
                               p.tiles};
  } else {
    p.prefix_tiles = P ? static_cast<int>((rows + 15) / 16) : 0;
  }
  p.prefix_units = (P + fa4d::kUnitKeys - 1) / fa4d::kUnitKeys;
  p.seg_rows = static_cast<int>(std::min<int64_t>(16, p.prefix_tiles ? rows : p.R));
  out->ctas = sms * (D == 256 ? fa4d::kDecodeCtas<256> : fa4d::kDecodeCtas<128>);
  p.min_units = 2;
  const int64_t items = static_cast<int64_t>(p.prefix_tiles) * Hk + static_cast<int64_t>(B) * Hk * p.tiles;
  if (items > (1 << 30)) return fail(FA4D_ERR_UNSUPPORTED, "too many row tiles");
  if (!out->splits) {
    // No more CTAs than full caches could occupy.
    const int64_t line = static_cast<int64_t>(p.prefix_tiles) * Hk * (p.prefix_units + fa4d::kPrefixItemUnits) +
                         static_cast<int64_t>(B) * Hk * p.tiles * ((C + fa4d::kUnitKeys - 1) / fa4d::kUnitKeys + fa4d::kItemUnits);
    const int64_t each = p.min_units * fa4d::kDecodeWarps;
    out->ctas = static_cast<int>(std::min<int64_t>(out->ctas, (line + each - 1) / each));
  }
  p.warps = out->ctas * fa4d::kDecodeWarps;
  p.logits_ld = (C + 3) / 4 * 4;
  const size_t seg = (static_cast<size_t>(items) + p.warps) * p.seg_rows;
  out->seg_o = 0;
  out->seg_ml = align256(seg * D * sizeof(float));
  out->logits = out->seg_ml + align256(seg * sizeof(float2));
  const size_t own_rows = weights ? static_cast<size_t>(B) * Hk * p.R : 0;
  out->lse = out->logits + align256(own_rows * p.logits_ld * sizeof(float));
  out->pre_o = out->lse + align256(own_rows * sizeof(float));
  const size_t pre = static_cast<size_t>(p.splits) * Hk * p.pre_rows;
  out->pre_ml = out->pre_o + align256(pre * D * sizeof(float));
  out->shares = out->pre_ml + align256(pre * sizeof(float2));
  out->total = out->shares + 256;
  return FA4D_OK;
}

}  // namespace

extern "C" {

int fa4d_rotary(const fa4d_rotary_args* a, void* stream) {
  if (!a) return fail(FA4D_ERR_INVALID, "args is NULL");
  int rc = check_table(a->table, a->positions_bits);
  if (!rc) rc = check_dtype(a->dtype);
  if (rc) return rc;
  if (!a->q || !a->k || !a->q_out || !a->k_out || !a->positions)
    return fail(FA4D_ERR_INVALID, "q, k, q_out, k_out and positions are required");
  if (a->B < 1 || a->T < 1 || a->Hq < 1 || a->Hk < 1 || a->Hq > (1 << 20) || a->Hk > (1 << 20))
    return fail(FA4D_ERR_INVALID, "sizes must be positive (B=%d T=%d Hq=%d Hk=%d)", a->B, a->T, a->Hq, a->Hk);
  if (static_cast<int64_t>(a->B) * a->T > (1LL << 31)) return fail(FA4D_ERR_UNSUPPORTED, "more than 2^31 tokens");
  if ((rc = host_bind_device_of(a->q, "q"))) return rc;
  const bool vec = table_vec(a->table) && rows16(a->q, a->q_stride, 3) && rows16(a->k, a->k_stride, 3) &&
                   rows16(a->q_out, a->q_out_stride, 3) && rows16(a->k_out, a->k_out_stride, 3);
  return launched(fa4d::launch_rotary(*a, vec, fa4d::host_sm_count(), static_cast<cudaStream_t>(stream)), "rotary");
}

int fa4d_rotary_append(const fa4d_rotary_append_args* a, void* stream) {
  if (!a) return fail(FA4D_ERR_INVALID, "args is NULL");
  int rc = check_table(a->table, a->positions_bits);
  if (!rc) rc = check_dtype(a->dtype);
  if (rc) return rc;
  if (!a->q || !a->k || !a->v || !a->q_out || !a->k_cache || !a->v_cache || !a->positions || !a->lengths ||
      !a->lengths_out)
    return fail(FA4D_ERR_INVALID, "q, k, v, q_out, the caches, positions, lengths and lengths_out are required");
  if (a->lengths == a->lengths_out) return fail(FA4D_ERR_INVALID, "lengths_out may not be lengths");
  if (a->B < 1 || a->T < 1 || a->Hq < 1 || a->Hk < 1 || a->C < 1)
    return fail(FA4D_ERR_INVALID, "sizes must be positive (B=%d T=%d Hq=%d Hk=%d C=%d)", a->B, a->T, a->Hq, a->Hk, a->C);
  if (static_cast<int64_t>(a->B) * a->T * (a->Hq + 2LL * a->Hk) > (1LL << 31))
    return fail(FA4D_ERR_UNSUPPORTED, "more than 2^31 rows");
  if ((rc = host_bind_device_of(a->q, "q"))) return rc;
  int* status = fa4d::host_status_word();
  if (!status) return fail(FA4D_ERR_CUDA, "device status word is not available");
  const bool vec = table_vec(a->table) && rows16(a->q, a->q_stride, 3) && rows16(a->k, a->k_stride, 3) &&
                   rows16(a->v, a->v_stride, 3) && rows16(a->q_out, a->q_out_stride, 3) &&
                   rows16(a->k_cache, a->k_cache_stride, 3) && rows16(a->v_cache, a->v_cache_stride, 3);
  return launched(fa4d::launch_rotary_append(*a, vec, status, static_cast<cudaStream_t>(stream)), "rotary append");
}

size_t fa4d_prefix_attention_workspace(int32_t B, int32_t T, int32_t Hq, int32_t Hk, int32_t D, int32_t P, int32_t C,
                                       int32_t weights) {
  Plan plan;
  return plan_prefix(B, T, Hq, Hk, D, P, C, weights != 0, &plan) ? 0 : plan.total;
}

int fa4d_prefix_attention(const fa4d_prefix_attention_args* a, void* stream) {
  if (!a) return fail(FA4D_ERR_INVALID, "args is NULL");
  int rc = check_dtype(a->dtype);
  if (rc) return rc;
  if (!a->q || !a->k || !a->v || !a->o || !a->lengths) return fail(FA4D_ERR_INVALID, "q, k, v, o and lengths are required");
  if ((a->P > 0) != (a->prefix_k != nullptr) || (a->P > 0) != (a->prefix_v != nullptr))
    return fail(FA4D_ERR_INVALID, "prefix_k and prefix_v go with P > 0");
  if (!std::isfinite(a->scale)) return fail(FA4D_ERR_INVALID, "scale is not finite");
  if (a->causal != 0 && a->causal != 1) return fail(FA4D_ERR_INVALID, "causal must be 0 or 1");
  if ((rc = host_bind_device_of(a->q, "q"))) return rc;
  Plan plan;
  if ((rc = plan_prefix(a->B, a->T, a->Hq, a->Hk, a->D, a->P, a->C, a->weights != nullptr, &plan))) return rc;
  if (!a->workspace || a->workspace_bytes < plan.total)
    return fail(FA4D_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", a->workspace_bytes, plan.total);
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0)
    return fail(FA4D_ERR_LAYOUT, "workspace must be 256-byte aligned");
  const struct {
    const void* p;
    const int64_t* st;
    int n;
    const char* name;
  } rows[] = {{a->q, a->q_stride, 3, "q"},
              {a->k, a->k_stride, 3, "k"},
              {a->v, a->v_stride, 3, "v"},
              {a->o, a->o_stride, 3, "o"},
              {a->prefix_k, a->prefix_k_stride, 2, "prefix_k"},
              {a->prefix_v, a->prefix_v_stride, 2, "prefix_v"}};
  for (const auto& r : rows)
    if (r.p && !rows16(r.p, r.st, r.n))
      return fail(FA4D_ERR_LAYOUT, "%s: rows must start on 16-byte boundaries", r.name);

  fa4d::DecodeParams& p = plan.p;
  char* ws = static_cast<char*>(a->workspace);
  p.q = a->q;
  p.o = a->o;
  p.lengths = a->lengths;
  p.mask = a->mask;
  p.weights = a->weights;
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = a->q_stride[i];
    p.o_stride[i] = a->o_stride[i];
    p.mask_stride[i] = a->mask_stride[i];
  }
  for (int i = 0; i < 2; ++i) p.weights_stride[i] = a->weights_stride[i];
  p.weights_vec = aligned16(a->weights) && a->weights_stride[0] % 4 == 0 && a->weights_stride[1] % 4 == 0;
  p.causal = a->causal;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.seg_o = reinterpret_cast<float*>(ws + plan.seg_o);
  p.seg_ml = reinterpret_cast<float2*>(ws + plan.seg_ml);
  p.logits = a->weights ? reinterpret_cast<float*>(ws + plan.logits) : nullptr;
  p.lse = reinterpret_cast<float*>(ws + plan.lse);
  p.pre_o = reinterpret_cast<float*>(ws + plan.pre_o);
  p.pre_ml = reinterpret_cast<float2*>(ws + plan.pre_ml);
  p.shares = reinterpret_cast<fa4d::Shares*>(ws + plan.shares);
  p.status = fa4d::host_status_word();
  if (!p.status) return fail(FA4D_ERR_CUDA, "device status word is not available");
  const bool bf16 = a->dtype == FA4D_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto encode = [&](CUtensorMap* m, const void* ptr, int B, int T, const int64_t st[3], int rows, const char* name) {
    return fa4d::host_encode_bthd(m, ptr, B, T, a->Hk, a->D, st, rows, bf16, name);
  };
  if ((rc = encode(&p.tm_k, a->k, a->B, a->C, a->k_stride, fa4d::kUnitKeys, "k"))) return rc;
  if ((rc = encode(&p.tm_v, a->v, a->B, a->C, a->v_stride, fa4d::kUnitKeys, "v"))) return rc;
  const int64_t ks[3] = {0, a->prefix_k_stride[0], a->prefix_k_stride[1]};
  const int64_t vs[3] = {0, a->prefix_v_stride[0], a->prefix_v_stride[1]};
  if (p.prefix_tiles) {
    if ((rc = encode(&p.tm_pk, a->prefix_k, 1, a->P, ks, fa4d::kUnitKeys, "prefix_k"))) return rc;
    if ((rc = encode(&p.tm_pv, a->prefix_v, 1, a->P, vs, fa4d::kUnitKeys, "prefix_v"))) return rc;
  }
  if (plan.splits) {
    fa4d::PrefixParams x;
    memset(&x, 0, sizeof(x));
    if ((rc = encode(&x.tm_k, a->prefix_k, 1, a->P, ks, 128, "prefix_k"))) return rc;
    if ((rc = encode(&x.tm_v, a->prefix_v, 1, a->P, vs, 128, "prefix_v"))) return rc;
    x.q = a->q;
    for (int i = 0; i < 3; ++i) x.q_stride[i] = a->q_stride[i];
    x.T = a->T;
    x.G = p.G;
    x.P = a->P;
    x.rows = p.pre_rows;
    x.parts = p.splits;
    x.d_in = a->D;
    x.lengths = a->lengths;
    x.B = a->B;
    x.C = a->C;
    x.Hk = a->Hk;
    x.load = p.load;
    x.shares = p.shares;
    x.scale_log2 = p.scale_log2;
    x.o = p.pre_o;
    x.ml = p.pre_ml;
    x.status = p.status;
    if ((rc = launched(fa4d::launch_prefix(x, a->D, bf16, a->Hk, plan.splits, plan.split_keys, s), "prefix attention")))
      return rc;
  }
  if ((rc = launched(fa4d::launch_decode(p, a->D, bf16, plan.ctas, plan.splits > 0, s), "decode attention"))) return rc;
  return launched(fa4d::launch_join(p, a->D, bf16, fa4d::host_sm_count(), s), "attention join");
}

int fa4d_evict(const fa4d_evict_args* a, void* stream) {
  if (!a) return fail(FA4D_ERR_INVALID, "args is NULL");
  if (!a->k || !a->v || !a->weights || !a->lengths || !a->k_out || !a->v_out || !a->weights_out || !a->lengths_out ||
      !a->index_out)
    return fail(FA4D_ERR_INVALID, "every pointer is required");
  if (a->B < 1 || a->C < 1 || a->Hk < 1 || a->D < 1 || a->keep < 1)
    return fail(FA4D_ERR_INVALID, "sizes must be positive (B=%d C=%d Hk=%d D=%d keep=%d)", a->B, a->C, a->Hk, a->D, a->keep);
  if (a->sinks < 0 || a->recent < 0 || static_cast<int64_t>(a->sinks) + a->recent > a->keep)
    return fail(FA4D_ERR_INVALID, "sinks (%d) and recent (%d) must fit in keep (%d)", a->sinks, a->recent, a->keep);
  if (static_cast<int64_t>(a->keep) * a->D > (1LL << 30) || a->C > (1 << 30) ||
      static_cast<int64_t>(a->B) * a->Hk > (1 << 27))
    return fail(FA4D_ERR_UNSUPPORTED, "cache too large (keep * D, C <= 2^30, B * Hk <= 2^27)");
  const void* in[] = {a->k, a->v, a->weights, a->lengths};
  const void* out[] = {a->k_out, a->v_out, a->weights_out, a->lengths_out};
  for (int i = 0; i < 4; ++i)
    if (in[i] == out[i]) return fail(FA4D_ERR_INVALID, "an output may not be an input");
  int rc = host_bind_device_of(a->k, "k");
  if (rc) return rc;
  const bool vec = a->D % 8 == 0 && rows16(a->k, a->k_stride, 3) && rows16(a->v, a->v_stride, 3) &&
                   rows16(a->k_out, a->k_out_stride, 3) && rows16(a->v_out, a->v_out_stride, 3);
  return launched(fa4d::launch_evict(*a, vec, fa4d::host_sm_count(), static_cast<cudaStream_t>(stream)), "evict");
}

}  // extern "C"
