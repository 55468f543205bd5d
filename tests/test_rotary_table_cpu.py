"""CPU: the rotary table against 60-digit arithmetic.

turn[i] = base^(-2 i / rotary_dim) / (2 pi) modulo 1, in units of 2^-64, worked out with 64-bit
mantissas.  For base >= 1 the turn is at most 0.16, so powl (an ulp, 2^-63) is off by 0.32 units,
the division by 0.16 and its constant by 0.08, the exponent's rounding by 0.06 (x e^-x <= 0.37);
rounding to nearest adds 0.5: at most 1.12 units, and as often too much as too little."""

from __future__ import annotations

from decimal import Decimal, getcontext

import pytest

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib

TWO_PI = Decimal("6.283185307179586476925286766559005768394338798750211641949889184615632812572417997256")


@pytest.mark.parametrize("base", [1.0, 10.0, 1e4, 5e5, 1e6])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_turns_are_rounded_to_nearest(base, dim):
    getcontext().prec = 60
    turns, _ = _lib.host().table_turns(api.MultiAxisRotary(dim, (dim // 2,), base=base)._table)
    off = []
    for i, turn in enumerate(turns):
        want = Decimal(base) ** (Decimal(-2 * i) / dim) / TWO_PI * 2 ** 64
        off.append(float(Decimal(turn) - want))
    assert max(map(abs, off)) <= 1.12
    if base > 1:  # 32 pairs or more: a mean of rounding errors is within 0.3, of truncation near -0.5
        assert abs(sum(off) / len(off)) < 0.3
