// fa4d_line.cuh — the line of units (fa4d_decode.h) as a warp walks it, for units of 2^kShift keys.
#pragma once

#include "fa4d_decode.h"
#include "fa4d_ptx.cuh"

namespace fa4d {

__device__ __forceinline__ int length_of(const DecodeParams& p, int b) { return length_at(p.lengths, b, p.C); }
// The division of `total` units.  Beside a prefix kernel the warps of the SMs that it leaves
// free start at once, and the others when it is done: those get less, by its estimated time.
template <int D>
__device__ __forceinline__ Shares shares_of(const DecodeParams& p, int64_t total, int lane) {
  const int least = p.min_units;
  auto up = [](int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); };
  if (p.load.items) {
    RunChoice c = choose_runs<D == 96 ? 128 : D>(p.load, total * p.heads, lane);
    c.rate /= p.heads;
    const int free_sms = p.load.sms - p.load.items * c.runs;
    if (free_sms > 0) {
      const int early = p.warps / p.load.sms * free_sms, rest = p.warps - early;
      // When all SMs work on the own keys; the late warps' part of that.
      const float late_us = fmaxf(c.total_us - c.prefix_us - kDecodeMicros, 0.f);
      const float part = fminf(late_us * c.rate * rest / p.warps, static_cast<float>(total));
      const int late = static_cast<int>(part / max(rest, 1));
      return Shares{early, max(up(total - static_cast<int64_t>(late) * rest, early), least), late, 0};
    }
  }
  return even_shares(total, p.warps, least);
}

__device__ __forceinline__ int64_t warp_start(const Shares& s, int64_t warp) {
  return min(warp, static_cast<int64_t>(s.early)) * s.each + max(warp - s.early, static_cast<int64_t>(0)) * s.late;
}
__device__ __forceinline__ int64_t warp_of(const Shares& s, int64_t unit) {
  const int64_t early = static_cast<int64_t>(s.early) * s.each;
  return unit < early ? quotient(unit, s.each) : s.early + quotient(unit - early, max(s.late, 1));
}

// The lengths of the first 128 requests in a warp's registers (lane l: l, l + 32, ...), the
// others in memory.
template <int kShift>
struct Lengths {
  int n[4];
  __device__ __forceinline__ void load(const DecodeParams& p, int lane) {
#pragma unroll
    for (int x = 0; x < 4; ++x) n[x] = length_of(p, min(32 * x + lane, p.B - 1));
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (32 * x + lane >= p.B) n[x] = 0;
  }
  __device__ __forceinline__ int of(const DecodeParams& p, int b) const {
    if (b >= 128) return length_of(p, b);
    return __shfl_sync(0xffffffffu, b < 64 ? (b < 32 ? n[0] : n[1]) : (b < 96 ? n[2] : n[3]), b & 31);
  }
  // What all requests take of the line, per KV head and row tile.
  __device__ __forceinline__ int64_t line(const DecodeParams& p, int lane) const {
    int64_t all = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) all += line_of(n[x], kShift);
    for (int i = 128 + lane; i < p.B; i += 32) all += line_of(length_of(p, i), kShift);
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    return all;
  }
};

// A place on the line, in a run with `left` of it to go.
template <int kShift>
struct Place {
  bool prefix;
  int b, hk, tile;  // the item (b unused in the prefix); hk: the group of heads
  int u, units;     // unit within the item, units of the item
  int keys;         // keys of the item
  int64_t left;

  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ int item(const DecodeParams& p) const {
    return prefix ? hk * p.prefix_tiles + tile : (p.prefix_tiles + b * p.tiles) * p.groups + hk * p.tiles + tile;
  }
  __device__ __forceinline__ void next_item(const DecodeParams& p, const Lengths<kShift>& lengths) {
    u = 0;
    if (++tile < (prefix ? p.prefix_tiles : p.tiles)) return;
    tile = 0;
    if (++hk < p.groups) return;
    hk = 0;
    b = prefix ? 0 : b + 1;
    prefix = false;
    for (; b < p.B; ++b) {  // the next request with keys
      keys = lengths.of(p, b);
      units = units_of(keys, kShift);
      if (units) return;
    }
    left = 0;
  }
  // To the next unit; true if it is of another item.
  __device__ __forceinline__ bool advance(const DecodeParams& p, const Lengths<kShift>& lengths) {
    --left;
    if (++u < units) return false;
    left -= prefix ? kPrefixItemUnits : kItemUnits;
    next_item(p, lengths);
    return true;
  }
};

// The first unit at or after `at` on the line, in a run of `left`.
template <int kShift>
__device__ __forceinline__ Place<kShift> find_place(const DecodeParams& p, const Lengths<kShift>& lengths, int64_t at, int64_t left,
                                            int lane) {
  Place<kShift> w;
  w.left = left;
  w.b = 0;
  int64_t line = p.prefix_units + kPrefixItemUnits;
  const int64_t prefix_all = static_cast<int64_t>(p.prefix_tiles) * p.groups * line;
  int tiles = p.tiles;
  w.prefix = at < prefix_all;
  if (w.prefix) {
    w.keys = p.P;
    tiles = p.prefix_tiles;
  } else {
    at -= prefix_all;
    const int64_t each = static_cast<int64_t>(p.groups) * p.tiles;
    bool found = false;
    auto search = [&](int b0, int mine) {  // among the 32 requests from b0
      int64_t upto = line_of(mine, kShift);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t before = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += before;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto * each > at);
      found = past != 0;
      const int l = found ? __ffs(past) - 1 : 31;
      const int64_t to = __shfl_sync(0xffffffffu, upto, l);
      if (!found) {
        at -= to * each;
        return;
      }
      w.b = b0 + l;
      w.keys = __shfl_sync(0xffffffffu, mine, l);
      line = line_of(w.keys, kShift);
      at -= (to - line) * each;
    };
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (!found && 32 * x < p.B) search(32 * x, lengths.n[x]);
    for (int b0 = 128; !found && b0 < p.B; b0 += 32)
      search(b0, b0 + lane < p.B ? length_of(p, b0 + lane) : 0);
  }
  w.units = units_of(w.keys, kShift);
  const int64_t item = at / line;
  w.hk = static_cast<int>(item / tiles);
  w.tile = static_cast<int>(item - static_cast<int64_t>(w.hk) * tiles);
  w.u = static_cast<int>(at - item * line);
  if (w.u >= w.units) {  // in the item's change of rows
    w.left -= line - w.u;
    w.next_item(p, lengths);
  }
  return w;
}

}  // namespace fa4d
