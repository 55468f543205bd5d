// fa4d_mma.cuh — the two tcgen05 products of an attention tile, shared by the forward kernel
// and the shared-prefix kernel.
#pragma once

#include "fa4d_ptx.cuh"

namespace fa4d {

// S[slot] = Q[slot] K^T : M=128, N=128, K=D; both operands K-major, 128-B swizzled.
template <int D, bool kBF16>
__device__ __forceinline__ void issue_qk(uint32_t tS, uint32_t sQ, uint32_t sK) {
  constexpr uint32_t idesc = make_idesc(128, 128, kBF16, false, false);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = static_cast<uint32_t>((kk >> 2) * 16384 + (kk & 3) * 32);
    mma_ss(tS, sw128_desc(sQ + off, 16, 1024), sw128_desc(sK + off, 16, 1024), idesc, kk > 0 ? 1u : 0u);
  }
}

// O[slot] (+)= P[slot] V : M=128, N=D, K=128; P from TMEM, V MN-major.  Covers keys
// [64 * first_half, 64 * last_half + 64) of the tile (K-steps of 16 keys).
template <int D, bool kBF16>
__device__ __forceinline__ void issue_pv(uint32_t tO, uint32_t tP, uint32_t sV, bool accumulate, int first_half = 0,
                                         int last_half = 1) {
  constexpr uint32_t idesc = make_idesc(128, D, kBF16, false, true);
#pragma unroll
  for (int kk = 4 * first_half; kk < 4 * last_half + 4; ++kk) {
    mma_ts(tO, tP + kk * 8, sw128_desc(sV + kk * 2048, 16384, 1024), idesc,
           (accumulate || kk > 0) ? 1u : 0u);
  }
}

}  // namespace fa4d
