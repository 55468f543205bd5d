"""What an entry's weight gains is summed over the rows before it is added.

Bound: the gain of R rows carries its own error (logits e = (D + 8) 2^-24 max sum|q k| |scale|
and 2^-19 for exponentials and sums of the softmax, R 2^-24 for the sum over the rows), and the
sum with what is there is rounded once: |w - (w0 + gain)| <= (2 e + 2^-19 + R 2^-24) gain +
2^-24 (w0 + gain)."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from oracle.serving import shared_prefix_ref

DEV = torch.device("cuda", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("start", [0.0, 100.0, 1e3, 1e4])
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", [
    (2, 1, 8, 1, 64, 0, 1100),  # 8 rows
    (1, 4, 16, 2, 128, 30, 70),  # 32
    (2, 4, 16, 1, 64, 0, 1500),  # 64
    (1, 9, 14, 1, 64, 300, 1030),  # 126: two batches of rows
    (1, 32, 8, 2, 128, 5, 600),  # 128
])
def test_many_rows_against_a_large_weight(B, T, Hq, Hk, D, P, C, start):
    g = torch.Generator().manual_seed(int(start) + T)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    q, k, v = r(B, Hq, T, D) * 0.25, r(B, Hk, C, D), r(B, Hk, C, D)
    pk, pv = (r(Hk, P, D), r(Hk, P, D)) if P else (None, None)
    lengths = torch.full((B,), C, dtype=torch.int32, device=DEV)
    w0 = start * (1 + torch.rand(B, Hk, C, generator=g).to(DEV)) / 2
    w = w0.clone()
    api.shared_prefix_attention(q, pk, pv, k, v, lengths, weights=w)
    _, gain, _, biggest = shared_prefix_ref(q, pk, pv, k, v, lengths)
    e = (D + 8) * 2.0 ** -24 * biggest
    R = T * Hq // Hk
    want = w0.double() + gain
    bound = (2 * e + 2.0 ** -19 + R * 2.0 ** -24) * gain + 2.0 ** -24 * want
    off = (w.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
