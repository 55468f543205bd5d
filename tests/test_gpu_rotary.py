"""Rotary positions with several axes against the 64-bit formula: forward, gradient,
appending to a cache.

Bound: the result is rounded once from 32 bits, whose own error (two products and a sum of
values up to |x|, angles to 2^-23) is below 2^-20 max|x|: |y - y64| <= u |y64| + 2^-20 max|x|
with u = 2^-8 (bf16) or 2^-11 (fp16), plus half the smallest fp16 step 2^-25."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.serving import rotary_ref

DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(y, ref, x):
    bound = U[y.dtype] * ref.abs() + 2.0 ** -20 * float(x.double().abs().max()) + 2.0 ** -25
    assert bool(((y.double() - ref).abs() <= bound).all()), float(((y.double() - ref).abs() - bound).max())


def tokens(g, B, H, T, D, dtype, layout):
    x = torch.randn((B, H, T, D) if layout == "bhsd" else (B, T, H, D), generator=g).to(dtype)
    return x.to(DEV)


CASES = [
    # (B, T, Hq, Hk, D, rotary_dim, sections, pairing, dtype, layout)
    (1, 1, 1, 1, 2, None, (1,), "half", torch.bfloat16, "bhsd"),
    (2, 5, 3, 1, 64, None, (8, 12, 12), "half", torch.bfloat16, "bhsd"),
    (1, 33, 8, 2, 128, None, (16, 24, 24), "adjacent", torch.float16, "bshd"),
    (2, 129, 5, 5, 96, 64, (10, 11, 11), "half", torch.float16, "bhsd"),
    (1, 17, 4, 2, 256, 96, (48,), "adjacent", torch.bfloat16, "bshd"),
    (3, 7, 2, 1, 80, 36, (9, 0, 9), "half", torch.bfloat16, "bshd"),  # no runs of 8
    (1, 300, 9, 3, 256, None, (32, 32, 32, 32), "half", torch.float16, "bshd"),
    (2, 11, 1, 3, 22, 10, (2, 3), "adjacent", torch.float16, "bhsd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,rot,sections,pairing,dtype,layout", CASES)
def test_forward_and_gradient_match_the_formula(B, T, Hq, Hk, D, rot, sections, pairing, dtype, layout):
    g = torch.Generator().manual_seed(B * 1000 + T)
    rope = api.MultiAxisRotary(D, sections, base=1e4, rotary_dim=rot, pairing=pairing)
    q, k = (tokens(g, B, H, T, D, dtype, layout).requires_grad_() for H in (Hq, Hk))
    pos = torch.randint(-50, 100000, (len(sections), B, T), generator=g, dtype=torch.int32).to(DEV)
    kw = dict(base=1e4, rotary_dim=rot, pairing=pairing, layout=layout)
    yq, yk = rope(q, k, pos, layout=layout)
    close(yq.detach(), rotary_ref(q.detach(), pos, sections, **kw), q.detach())
    close(yk.detach(), rotary_ref(k.detach(), pos, sections, **kw), k.detach())
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    close(gq, rotary_ref(dq, pos, sections, inverse=True, **kw), dq)
    close(gk, rotary_ref(dk, pos, sections, inverse=True, **kw), dk)
    # Without autograd, with 64-bit and broadcast positions: the same bits.
    with torch.no_grad():
        again = rope(q, k, pos.long(), layout=layout)
        assert torch.equal(again[0], yq) and torch.equal(again[1], yk)
        one = rope(q, k, pos[:, :1], layout=layout)
        each = rope(q, k, pos[:, :1].expand(-1, B, -1).contiguous(), layout=layout)
        assert torch.equal(one[0], each[0]) and torch.equal(one[1], each[1])


@pytest.mark.gpu
def test_gradient_matches_differences():
    """The op is linear in q, so f(q + e d) - f(q - e d) over 2 e is its derivative along d up
    to rounding: <dy, that> = <grad, d>.  Each side sums N = 2 * 6 * 3 * 64 products of rounded
    values; with e = 1 and unit normals the rounding of y (2^-11 each) gives both sides a
    standard error of about 2^-11 sqrt(N); eight of them are allowed."""
    g = torch.Generator().manual_seed(3)
    rope = api.MultiAxisRotary(64, (8, 12, 12))
    q, d = tokens(g, 2, 3, 6, 64, torch.float16, "bhsd"), tokens(g, 2, 3, 6, 64, torch.float16, "bhsd")
    pos = torch.randint(0, 999, (3, 2, 6), generator=g).to(DEV)
    dy = tokens(g, 2, 3, 6, 64, torch.float16, "bhsd")
    x = q.clone().requires_grad_()
    y, _ = rope(x, q, pos)
    (grad,) = torch.autograd.grad(y, x, dy)
    up, down = rope(q + d, q, pos)[0], rope(q - d, q, pos)[0]
    along = ((up.double() - down.double()) / 2 * dy.double()).sum()
    n = q.numel()
    assert abs(float(along - (grad.double() * d.double()).sum())) <= 8 * 2.0 ** -11 * n ** 0.5 * 2


@pytest.mark.gpu
def test_far_positions_lose_nothing():
    """Positions near 2^40, whose 32-bit product with a frequency would be off by many turns.
    The 64-bit reference itself has phi to 2^-12 there, so the fixed-point angle is compared
    through a base of 1 (every pair turns one radian a position): phi mod 2 pi from Python's
    integers and a 100-digit pi."""
    two_pi_scaled = 6283185307179586476925286766559005768394338798750211641949889184615632812572417997256069650684234135
    pos = torch.tensor([[[2 ** 40 + 12345, 2 ** 40 - 1, -(2 ** 39) - 7]]])
    exact = torch.tensor([((int(p) * 10 ** 99) % two_pi_scaled) / 10 ** 99 for p in pos.flatten()], dtype=torch.float64)
    # turn is exact to 2^-64 turns: 2^41 positions bring that to 2^-23; the rest is fp16's rounding.
    x = torch.zeros(1, 1, 3, 2, dtype=torch.float16)
    x[..., 0] = 1.0
    y, _ = api.MultiAxisRotary(2, (1,), base=1.0)(x.to(DEV), x.to(DEV), pos.to(DEV))
    y = y.cpu().double()[0, 0]
    assert float((y[:, 0] - exact.cos()).abs().max()) <= 2 ** -10 and float((y[:, 1] - exact.sin()).abs().max()) <= 2 ** -10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strided_and_unaligned_inputs_give_the_same_bits(dtype):
    g = torch.Generator().manual_seed(5)
    rope = api.MultiAxisRotary(64, (8, 12, 12))
    pos = torch.randint(0, 5000, (3, 2, 9), generator=g).to(DEV)
    q, k = tokens(g, 2, 4, 9, 64, dtype, "bhsd"), tokens(g, 2, 2, 9, 64, dtype, "bhsd")
    want = rope(q, k, pos)
    pad = torch.empty(2 * 4 * 9 * 64 + 1, dtype=dtype, device=DEV)
    odd = pad[1:].view(2, 4, 9, 64)  # 2 bytes past a 16-byte boundary
    odd.copy_(q)
    wide = torch.empty(2, 2, 9, 80, dtype=dtype, device=DEV)
    wide[..., 3:67].copy_(k)
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)  # head-dim stride 9
    for a, b in ((odd, k), (q, wide[..., 3:67]), (turned, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k)):
        got = rope(a, b, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same = rope(q[:, :1].expand(-1, 4, -1, -1), k, pos)  # one head for all
    assert torch.equal(same[0], rope(q[:, :1].repeat(1, 4, 1, 1), k, pos)[0])
    # Positions with strides of their own.
    assert torch.equal(rope(q, k, pos.permute(2, 1, 0).contiguous().permute(2, 1, 0))[0], want[0])


@pytest.mark.gpu
def test_infinities_stay_in_their_pair():
    rope = api.MultiAxisRotary(64, (32,))
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 0, 0, 5] = float("inf")
    x[0, 0, 1, 40] = float("nan")
    y, _ = rope(x, x, torch.zeros(1, 1, 2, dtype=torch.int64, device=DEV))
    bad = ~torch.isfinite(y[0, 0])
    assert bad[0].nonzero().flatten().tolist() == [5, 37] and bad[1].nonzero().flatten().tolist() == [8, 40]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,rot,sections,pairing,dtype,layout", CASES)
def test_append(B, T, Hq, Hk, D, rot, sections, pairing, dtype, layout):
    g = torch.Generator().manual_seed(T)
    C = T + 9
    rope = api.MultiAxisRotary(D, sections, rotary_dim=rot, pairing=pairing)
    q, k, v = (tokens(g, B, H, T, D, dtype, layout) for H in (Hq, Hk, Hk))
    kc, vc = (tokens(g, B, Hk, C, D, dtype, layout) for _ in range(2))
    w = torch.rand(B, Hk, C, generator=g).to(DEV)
    lengths = torch.randint(0, 10, (B,), generator=g, dtype=torch.int32).to(DEV)
    pos = torch.randint(0, 9999, (len(sections), B, T), generator=g).to(DEV)
    want_q, want_k = rope(q, k, pos, layout=layout)
    want = [kc.clone(), vc.clone(), w.clone()]
    for b in range(B):
        n = int(lengths[b])
        at = (b, slice(None), slice(n, n + T)) if layout == "bhsd" else (b, slice(n, n + T))
        want[0][at], want[1][at] = want_k[b], v[b]
        want[2][b, :, n:n + T] = 0
    got_q, new = rope.append(q, k, v, pos, kc, vc, lengths, weights=w, layout=layout)
    assert torch.equal(got_q, want_q) and torch.equal(new, lengths + T)
    for a, b in zip((kc, vc, w), want):
        assert torch.equal(a, b)
    assert _lib.device_status(DEV) == 0


@pytest.mark.gpu
def test_append_to_a_full_cache_stores_what_fits_and_says_so():
    rope = api.MultiAxisRotary(64, (32,))
    x = torch.ones(2, 1, 3, 64, dtype=torch.bfloat16, device=DEV)
    kc, vc = torch.zeros(2, 1, 5, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 1, 5, 64, dtype=torch.bfloat16, device=DEV)
    lengths = torch.tensor([4, 1], dtype=torch.int32, device=DEV)
    _, new = rope.append(x, x, x, torch.zeros(1, 1, 3, dtype=torch.int32, device=DEV), kc, vc, lengths)
    assert new.tolist() == [5, 4]
    assert vc[..., 0].int().tolist() == [[[0, 0, 0, 0, 1]], [[0, 1, 1, 1, 0]]]
    assert _lib.device_status(DEV) == _lib.DEV_CACHE_FULL
    assert _lib.device_status(DEV) == 0


@pytest.mark.gpu
def test_empty_and_other_stream():
    rope = api.MultiAxisRotary(64, (32,))
    for shape, pos in (((0, 2, 3, 64), (1, 0, 3)), ((2, 2, 0, 64), (1, 2, 0))):
        x = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        y, _ = rope(x, x, torch.empty(pos, dtype=torch.int64, device=DEV))
        assert y.shape == x.shape
    x = torch.randn(1, 2, 4096, 64, device=DEV).bfloat16()
    pos = torch.arange(4096, device=DEV)[None, None]
    want = rope(x, x, pos)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = x * 1  # made on the side stream just before the call
        got = rope(z, z, pos)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows of the last request lie past 2^31 elements."""
    store = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device=DEV)
    big = store.as_strided((2, 1, 4, 64), (2 ** 31 + 8, 256, 64, 1))
    g = torch.Generator().manual_seed(0)
    q = tokens(g, 2, 1, 4, 64, torch.bfloat16, "bhsd")
    big.copy_(q)
    pos = torch.arange(8, device=DEV).view(1, 2, 4)
    rope = api.MultiAxisRotary(64, (32,))
    want, _ = rope(q, q, pos)
    got, _ = rope(big, q, pos)
    assert torch.equal(got, want)
    store.zero_()
    rope.append(q, q, q, pos, big, q.clone(), torch.zeros(2, dtype=torch.int32, device=DEV))
    assert torch.equal(big, want)
