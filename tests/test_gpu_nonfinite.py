"""Attention over a shared prefix and own caches where values have diverged: a row that sees a
NaN or an undefined softmax is NaN, as in the formula, and no other row changes by a bit."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.serving import shared_prefix_ref

DEV = torch.device("cuda", 0)
NAN, INF = float("nan"), float("inf")

# (B, T, Hq, Hk, D, P, C): the decode kernel alone, with the prefix too, then the prefix kernel
# with both slots on the same rows, with 256 rows, and at head dim 256; few rows (several warps of
# the join take one) and many; more than 32 rows of a KV head (the weights take their sums from the
# join) and fewer.
SIZES = [
    (3, 1, 4, 2, 64, 0, 40),
    (3, 2, 8, 2, 128, 70, 300),
    (150, 1, 16, 2, 64, 0, 33),
    (2, 12, 8, 2, 96, 40, 50),
    (4, 2, 8, 2, 256, 90, 40),
    (12, 1, 16, 2, 64, 6001, 20),
    (40, 1, 8, 1, 128, 4200, 60),
    (20, 2, 8, 2, 128, 3000, 1100),
    (16, 2, 4, 2, 256, 2177, 30),
]


def make(B, T, Hq, Hk, D, P, C, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed + B + P)
    r = lambda *s: torch.randn(s, generator=g).to(dtype).to(DEV)  # noqa: E731
    lengths = torch.randint(T, C + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
    return r(B, Hq, T, D), (r(Hk, P, D) if P else None), (r(Hk, P, D) if P else None), r(B, Hk, C, D), r(B, Hk, C, D), lengths


def attend(q, pk, pv, k, v, lengths, **kw):
    w = torch.zeros(k.shape[:3], device=DEV)
    out = api.shared_prefix_attention(q, pk, pv, k, v, lengths, weights=w, **kw)
    plain = api.shared_prefix_attention(q, pk, pv, k, v, lengths, **kw)
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))
    assert _lib.device_status(DEV) == 0
    return out, w


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", SIZES)
def test_a_nan_query_row_is_nan_and_no_other(B, T, Hq, Hk, D, P, C):
    q, pk, pv, k, v, lengths = make(B, T, Hq, Hk, D, P, C)
    want, want_w = attend(q, pk, pv, k, v, lengths)
    b, h, t = B - 1, Hq - 1, 0
    q = q.clone()
    q[b, h, t, 3] = NAN
    out, w = attend(q, pk, pv, k, v, lengths)
    assert bool(out[b, h, t].isnan().all())
    out[b, h, t] = want[b, h, t]
    assert torch.equal(out, want)
    # Its weights: NaN at the slots that it sees, the others as they were.
    sees = torch.zeros_like(w, dtype=torch.bool)
    sees[b, h * Hk // Hq, : int(lengths[b]) - T + t + 1] = True
    assert torch.equal(w.isnan(), sees)
    assert torch.equal(w[~sees], want_w[~sees])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", SIZES)
def test_a_nan_key_reaches_the_rows_that_see_it(B, T, Hq, Hk, D, P, C):
    """One own key, so that it is a part by itself beside the prefix."""
    q, pk, pv, k, v, lengths = make(B, T, Hq, Hk, D, P, C)
    lengths[B - 1] = T
    want, _ = attend(q, pk, pv, k, v, lengths)
    k = k.clone()
    k[B - 1, Hk - 1, 0, 5] = NAN
    out, _ = attend(q, pk, pv, k, v, lengths)
    G = Hq // Hk
    assert bool(out[B - 1, Hq - G :].isnan().all())
    out[B - 1, Hq - G :] = want[B - 1, Hq - G :]
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", [s for s in SIZES if s[5]])
def test_a_nan_prefix_key_reaches_every_row_of_its_head(B, T, Hq, Hk, D, P, C):
    q, pk, pv, k, v, lengths = make(B, T, Hq, Hk, D, P, C)
    want, _ = attend(q, pk, pv, k, v, lengths)
    pk = pk.clone()
    pk[0] = NAN
    out, _ = attend(q, pk, pv, k, v, lengths)
    G = Hq // Hk
    assert bool(out[:, :G].isnan().all()) and torch.equal(out[:, G:], want[:, G:])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", SIZES)
def test_an_infinite_query(B, T, Hq, Hk, D, P, C, value):
    """Keys that are positive where the query is infinite: every logit of the row is the same
    infinity, and its softmax undefined, not a row without a key."""
    q, pk, pv, k, v, lengths = make(B, T, Hq, Hk, D, P, C)
    b, h, t = B // 2, 0, T - 1
    for x in (k, pk):
        if x is not None:
            x[..., 3] = x[..., 3].abs() + 0.5
    want, _ = attend(q, pk, pv, k, v, lengths)
    q = q.clone()
    q[b, h, t, 3] = value
    out, _ = attend(q, pk, pv, k, v, lengths)
    assert bool(out[b, h, t].isnan().all())
    out[b, h, t] = want[b, h, t]
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [0, 9])
def test_rows_without_a_key_stay_zero_beside_diverged_ones(P):
    """A row whose mask leaves nothing is 0 (without a prefix) whatever its query holds, and a key
    of logit -inf counts as 0 where another is finite.  NaN and zero rows are the oracle's."""
    q, pk, pv, k, v, _ = make(2, 3, 4, 2, 64, P, 21)
    q[0, 1, 1] = NAN
    q[1, 2, 0, 7], q[1, 3, 2, 7] = INF, -INF
    k[:, :, 2:, 7] = k[:, :, 2:, 7].abs() + 0.5
    k[0, 0, 4, 7] = -INF
    q[0, :2, :, 7] = 1.0  # k[0, 0, 4] has logit -inf
    mask = torch.ones(2, 4, 3, 21, dtype=torch.bool, device=DEV)
    mask[:, :, 1] = False
    mask[:, :, :, :2] = False
    lengths = torch.tensor([21, 17], dtype=torch.int32, device=DEV)
    ref, _, _, _ = shared_prefix_ref(q, pk, pv, k, v, lengths, mask=mask)
    out, _ = attend(q, pk, pv, k, v, lengths, mask=mask)
    assert torch.equal(out.isnan(), ref.isnan())
    fine = ~ref.isnan()
    assert float((out.double() - ref)[fine].abs().max()) < 0.05
    if P == 0:
        assert not out[:, :, 1].any()
