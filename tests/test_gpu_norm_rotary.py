"""Norms of queries and keys with the rotary turn in the same pass, against the 64-bit formula:
forward, gradients, and the serving form with 16-bit caches.

Forward: n = x r w in 32 bits is off by at most (D + 16) 2^-24 of itself (a sum of D squares, the
reciprocal root, three products), the turn by 2^-20 max|n| (two products, a sum, angles to 2^-23),
and the result is rounded once: |y - y64| <= u |y64| + ((D + 16) 2^-24 + 2^-20) max|n| + 2^-25, the
last for fp16's smallest step; u = 2^-8 (bf16) or 2^-11 (fp16).

Gradient of x: with xh = x r, both terms of r (w g - xh mean(w g xh)) are off by at most
f = 2 (D + 64) 2^-24 + 2^-19 of their sizes with |g| replaced by its row's maximum (its turn's error
is relative to that): |dx - dx64| <= u |dx64| + f r G (max|w| + |xh| mean(|w xh|)) + 2^-25.
Gradient of w: N terms are off by f of G |xh| each and summed in 32 bits in chains of at most N:
(f + N 2^-24) sum G |xh|, and one rounding to the weights' type."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import norm_ref, norm_rotary_grads
from oracle.serving import rotary_ref

DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def tokens(g, B, H, T, D, dtype, layout, scale=1.0):
    x = torch.randn((B, H, T, D) if layout == "bhsd" else (B, T, H, D), generator=g) * scale
    return x.to(dtype).to(DEV)


def weights(g, D, dtype):
    return [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(DEV) for _ in range(2)]


def close(got, ref, bound):
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


def forward_close(y, x, w, pos, sections, eps, **kw):
    n = norm_ref(x, w, eps)
    ref, D = rotary_ref(n, pos, sections, **kw), x.shape[-1]
    close(y, ref, U[y.dtype] * ref.abs() + ((D + 16) * 2.0 ** -24 + 2.0 ** -20) * float(n.abs().max()) + 2.0 ** -25)


def gradients_close(dx, dw, x, w, dy, pos, sections, eps, **kw):
    g, rx, rw = norm_rotary_grads(x, w, dy, pos, sections, eps=eps, **kw)
    x, w, D = x.double(), w.double(), x.shape[-1]
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    xh, G = x * r, dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
    f = 2 * (D + 64) * 2.0 ** -24 + 2.0 ** -19
    size = r * G * (w.abs().max() + xh.abs() * (w * xh).abs().mean(-1, keepdim=True))
    close(dx, rx, U[dx.dtype] * rx.abs() + f * size + 2.0 ** -25)
    N = x.numel() // D
    close(dw, rw, U[dw.dtype] * rw.abs() + (f + N * 2.0 ** -24) * (G * xh.abs()).sum((0, 1, 2)) + 2.0 ** -25)


CASES = [
    # (B, T, Hq, Hk, D, rotary_dim, sections, pairing, dtype, weight dtype, layout)
    (1, 1, 1, 1, 2, None, (1,), "half", torch.bfloat16, torch.float32, "bhsd"),
    (2, 5, 3, 1, 64, None, (8, 12, 12), "half", torch.bfloat16, torch.bfloat16, "bhsd"),
    (1, 33, 8, 2, 128, None, (16, 24, 24), "adjacent", torch.float16, torch.float32, "bshd"),
    (2, 129, 5, 5, 96, 64, (10, 11, 11), "half", torch.float16, torch.float16, "bhsd"),
    (1, 17, 4, 2, 256, 96, (48,), "adjacent", torch.bfloat16, torch.float32, "bshd"),
    (3, 7, 2, 1, 80, 36, (9, 0, 9), "half", torch.bfloat16, torch.bfloat16, "bshd"),  # no runs of 8
    (1, 300, 9, 3, 256, None, (32, 32, 32, 32), "half", torch.float16, torch.float16, "bshd"),
    (2, 11, 1, 3, 22, 10, (2, 3), "adjacent", torch.float16, torch.float32, "bhsd"),
    (1, 700, 40, 7, 16, None, (4, 4), "half", torch.bfloat16, torch.float32, "bhsd"),
    (2, 1500, 28, 4, 32, 16, (8,), "adjacent", torch.float16, torch.float32, "bshd"),
]


def make(B, T, Hq, Hk, D, rot, sections, pairing, dtype, wide, layout):
    g = torch.Generator().manual_seed(B * 1000 + T)
    rope = api.MultiAxisRotary(D, sections, base=1e4, rotary_dim=rot, pairing=pairing)
    q, k = tokens(g, B, Hq, T, D, dtype, layout, 2.0), tokens(g, B, Hk, T, D, dtype, layout, 0.3)
    pos = torch.randint(-50, 100000, (len(sections), B, T), generator=g, dtype=torch.int32).to(DEV)
    return g, rope, q, k, pos, weights(g, D, wide), dict(base=1e4, rotary_dim=rot, pairing=pairing, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients_match_the_formula(case):
    layout, sections, eps = case[10], case[6], 1e-5
    g, rope, q, k, pos, (wq, wk), kw = make(*case)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    yq, yk = rope(q, k, pos, query_norm=wq, key_norm=wk, eps=eps, layout=layout)
    for y, x, w in ((yq, q, wq), (yk, k, wk)):
        forward_close(y.detach(), x.detach(), w.detach(), pos, sections, eps, **kw)
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    gq, gk, gwq, gwk = torch.autograd.grad((yq, yk), leaves, (dq, dk), retain_graph=True)
    gradients_close(gq, gwq, q.detach(), wq.detach(), dq, pos, sections, eps, **kw)
    gradients_close(gk, gwk, k.detach(), wk.detach(), dk, pos, sections, eps, **kw)
    assert gwq.dtype == wq.dtype and gq.dtype == q.dtype
    # The same bits every time, and without autograd, with 64-bit and broadcast positions.
    again = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(again, (gq, gk, gwq, gwk)))
    with torch.no_grad():
        plain = rope(q, k, pos.long(), query_norm=wq, key_norm=wk, eps=eps, layout=layout)
        assert torch.equal(plain[0], yq) and torch.equal(plain[1], yk)


@pytest.mark.gpu
def test_gradient_matches_differences():
    """<dy, (f(x + d) - f(x - d)) / 2> = <dx, d> + what the step leaves out, which the 64-bit formula
    gives.  With N values rounded by at most 2^-11 |y| on each side, |y| <= 8: eight standard errors
    of 2^-11 |y| |dy|, and of the gradient's own rounding, are below 8 * 2^-11 * 4 sqrt(N)."""
    g = torch.Generator().manual_seed(3)
    rope = api.MultiAxisRotary(64, (8, 12, 12))
    q, dy = tokens(g, 2, 3, 6, 64, torch.float16, "bhsd"), tokens(g, 2, 3, 6, 64, torch.float16, "bhsd")
    step = tokens(g, 2, 3, 6, 64, torch.float16, "bhsd", 0.1)
    pos = torch.randint(0, 999, (3, 2, 6), generator=g).to(DEV)
    w, dw = (x.half() for x in weights(g, 64, torch.float32))
    dw = dw * 0.1
    f = lambda x, w: rope(x, q, pos, query_norm=w, key_norm=w)[0]  # noqa: E731
    exact = lambda x, w: rotary_ref(norm_ref(x, w, 1e-6), pos, (8, 12, 12), base=1e4)  # noqa: E731
    x, v = q.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(f(x, v), (x, v), dy)
    _, ex, ew = norm_rotary_grads(q, w, dy, pos, (8, 12, 12), eps=1e-6, base=1e4)
    for (a, b), grad, ref in (((q + step, q - step), gx, ex), ((w + dw, w - dw), gw, ew)):
        d = (a.double() - b.double()) / 2
        both = [(i, w) if grad is gx else (q, i) for i in (a, b)]
        along = ((f(*both[0]).double() - f(*both[1]).double()) / 2 * dy.double()).sum()
        left_out = ((exact(*both[0]) - exact(*both[1])) / 2 * dy.double()).sum() - (ref * d).sum()
        assert abs(float(along - (grad.double() * d).sum() - left_out)) <= 8 * 2.0 ** -11 * 4 * q.numel() ** 0.5
        # And the formula against differences of itself, which leave out less.
        h = d * 1e-4
        ends = [exact(q + s * h, w) if grad is gx else exact(q, w + s * h) for s in (1, -1)]
        assert abs(float(((ends[0] - ends[1]) / 2 * dy.double()).sum() - (ref * h).sum())) <= 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strided_unaligned_and_shared_inputs(dtype):
    """Rows off 16-byte boundaries are taken pair by pair, in another order of the squares: within
    the formula's bound, as the strided views, whose bits are the same."""
    g = torch.Generator().manual_seed(5)
    rope = api.MultiAxisRotary(64, (8, 12, 12))
    pos = torch.randint(0, 5000, (3, 2, 9), generator=g).to(DEV)
    q, k = tokens(g, 2, 4, 9, 64, dtype, "bhsd"), tokens(g, 2, 2, 9, 64, dtype, "bhsd")
    wq, wk = weights(g, 64, torch.float32)
    kw = dict(query_norm=wq, key_norm=wk)
    want = rope(q, k, pos, **kw)
    pad = torch.empty(2 * 4 * 9 * 64 + 1, dtype=dtype, device=DEV)
    odd = pad[1:].view(2, 4, 9, 64)  # 2 bytes past a 16-byte boundary
    odd.copy_(q)
    forward_close(rope(odd, k, pos, **kw)[0], q, wq, pos, (8, 12, 12), 1e-6, base=1e4)
    wide = torch.zeros(2, 4, 9, 80, dtype=dtype, device=DEV)
    wide[..., 8:72].copy_(q)
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)  # head-dim stride 9
    for a in (wide[..., 8:72], turned, q.transpose(1, 2).contiguous().transpose(1, 2)):
        got = rope(a, k, pos, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # Weights with a stride, and one head or one request for all: their gradients add up.
    every = torch.stack([wq, wk], 1).flatten()[::2]
    assert torch.equal(rope(q, k, pos, query_norm=every, key_norm=wk)[0], want[0])
    one = q[:1, :1].clone().requires_grad_()
    w = wq.clone().requires_grad_()
    y, _ = rope(one.expand(2, 4, -1, -1), k, pos, query_norm=w, key_norm=w)
    dy = torch.randn_like(y)
    d1, dw = torch.autograd.grad(y, (one, w), dy)
    full = q[:1, :1].expand(2, 4, -1, -1).contiguous().requires_grad_()
    v = wq.clone().requires_grad_()
    d2, dv = torch.autograd.grad(rope(full, k, pos, query_norm=v, key_norm=v)[0], (full, v), dy)
    assert torch.equal(dw, dv) and torch.equal(d1, d2.sum((0, 1), keepdim=True, dtype=torch.float32).to(dtype)) or \
        float((d1.float() - d2.float().sum((0, 1), keepdim=True)).abs().max()) <= 8 * U[dtype] * 8 * float(d2.abs().max())


@pytest.mark.gpu
def test_gradients_with_strides_of_their_own_and_only_some_wanted():
    g = torch.Generator().manual_seed(6)
    rope = api.MultiAxisRotary(64, (32,))
    q, k = tokens(g, 2, 4, 9, 64, torch.bfloat16, "bhsd"), tokens(g, 2, 2, 9, 64, torch.bfloat16, "bhsd")
    pos = torch.arange(9, device=DEV).expand(1, 2, 9)
    wq, wk = weights(g, 64, torch.bfloat16)
    w = wq.clone().requires_grad_()
    y, yk = rope(q, k, pos, query_norm=w, key_norm=wk)
    assert yk.requires_grad  # one node has both outputs
    a, = torch.autograd.grad(y.sum(), w, retain_graph=True)  # a gradient of stride 0
    b, = torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)
    c, = torch.autograd.grad(y, w, torch.ones_like(y).transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(a, b) and torch.equal(b, c)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    rope = api.MultiAxisRotary(64, (32,))
    x = torch.randn(1, 2, 4, 64, device=DEV).bfloat16().requires_grad_()
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, _ = rope(x, x, torch.zeros(1, 1, 4, dtype=torch.int64, device=DEV), query_norm=w, key_norm=w)
    first, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(first.float().sum(), x)


@pytest.mark.gpu
def test_zeros_infinities_and_nan_stay_in_their_row():
    rope = api.MultiAxisRotary(64, (32,))
    x = torch.ones(1, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 0, 0] = 0
    x[0, 0, 1, 5] = float("inf")
    x[0, 0, 2, 40] = float("nan")
    x.requires_grad_()
    w = torch.ones(64, device=DEV)
    y, _ = rope(x, x, torch.zeros(1, 1, 4, dtype=torch.int64, device=DEV), query_norm=w, key_norm=w)
    bad = ~torch.isfinite(y[0, 0])
    assert not bad[0].any() and not y[0, 0, 0].any() and bad[1].any() and bad[2].all() and not bad[3].any()
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    bad = ~torch.isfinite(gx[0, 0])
    assert not bad[0].any() and bad[2].all() and not bad[3].any()


@pytest.mark.gpu
def test_empty_other_stream_and_graph():
    rope = api.MultiAxisRotary(64, (32,))
    w = torch.ones(64, device=DEV, requires_grad=True)
    for shape, pos in (((0, 2, 3, 64), (1, 0, 3)), ((2, 2, 0, 64), (1, 2, 0))):
        x = torch.empty(shape, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        y, _ = rope(x, x, torch.empty(pos, dtype=torch.int64, device=DEV), query_norm=w, key_norm=w)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape == gx.shape and not gw.any()
    g = torch.Generator().manual_seed(1)
    x, dy = tokens(g, 1, 2, 4096, 64, torch.bfloat16, "bhsd"), tokens(g, 1, 2, 4096, 64, torch.bfloat16, "bhsd")
    pos = torch.arange(4096, device=DEV)[None, None]

    def step(x):
        x = x.detach().requires_grad_()
        v = w.detach().requires_grad_()
        y, _ = rope(x, x, pos, query_norm=v, key_norm=v)
        return (y.detach(), *torch.autograd.grad(y, (x, v), dy))

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x * 1)  # made on the side stream just before the call
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, static = torch.cuda.CUDAGraph(), torch.zeros_like(x)
    step(static)
    with torch.cuda.graph(graph):
        got = step(static)
    static.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows of the last request lie past 2^31 elements, in every tensor."""
    g = torch.Generator().manual_seed(0)
    far = lambda: torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device=DEV).as_strided((2, 1, 4, 64), (2 ** 31 + 8, 256, 64, 1))  # noqa: E731
    q, dy = tokens(g, 2, 1, 4, 64, torch.bfloat16, "bhsd"), tokens(g, 2, 1, 4, 64, torch.bfloat16, "bhsd")
    big, big_dy = far(), far()
    big.copy_(q)
    big_dy.copy_(dy)
    pos = torch.arange(8, device=DEV).view(1, 2, 4)
    w = torch.ones(64, device=DEV)
    rope = api.MultiAxisRotary(64, (32,))
    results = []
    for x, d in ((q, dy), (big, big_dy)):
        x = x.detach().requires_grad_()
        y, _ = rope(x, q, pos, query_norm=w, key_norm=w)
        results.append((y.detach(), *torch.autograd.grad(y, x, d)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_append_to_16_bit_caches(case):
    B, T, Hq, Hk, D, rot, sections, pairing, dtype, wide, layout = case
    g, rope, q, k, pos, (wq, wk), kw = make(*case)
    C = T + 9
    v = tokens(g, B, Hk, T, D, dtype, layout)
    kc, vc = (tokens(g, B, Hk, C, D, dtype, layout) for _ in range(2))
    w = torch.rand(B, Hk, C, generator=g).to(DEV)
    lengths = torch.randint(0, 10, (B,), generator=g, dtype=torch.int32).to(DEV)
    had = [x.clone() for x in (kc, vc, w)]
    got_q, new = rope.append(q, k, v, pos, kc, vc, lengths, weights=w, query_norm=wq, key_norm=wk, eps=1e-5, layout=layout)
    assert torch.equal(new, lengths + T)
    forward_close(got_q, q, wq, pos, sections, 1e-5, **kw)
    stored = torch.empty_like(k)
    for b in range(B):
        n = int(lengths[b])
        at = (b, slice(None), slice(n, n + T)) if layout == "bhsd" else (b, slice(n, n + T))
        stored[b] = kc[at]
        had[0][at], had[1][at] = kc[at], v[b]
        had[2][b, :, n:n + T] = 0
    forward_close(stored, k, wk, pos, sections, 1e-5, **kw)
    for a, b in zip((kc, vc, w), had):
        assert torch.equal(a, b)
    assert _lib.device_status(DEV) == 0


@pytest.mark.gpu
def test_append_to_a_full_16_bit_cache():
    rope = api.MultiAxisRotary(64, (32,))
    x = torch.ones(2, 1, 3, 64, dtype=torch.bfloat16, device=DEV)
    kc, vc = torch.zeros(2, 1, 5, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 1, 5, 64, dtype=torch.bfloat16, device=DEV)
    lengths, w = torch.tensor([4, 1], dtype=torch.int32, device=DEV), torch.ones(64, device=DEV)
    _, new = rope.append(x, x, x, torch.zeros(1, 1, 3, dtype=torch.int32, device=DEV), kc, vc, lengths, query_norm=w, key_norm=w)
    assert new.tolist() == [5, 4]
    assert vc[..., 0].int().tolist() == [[[0, 0, 0, 0, 1]], [[0, 1, 1, 1, 0]]]
    assert _lib.device_status(DEV) == _lib.DEV_CACHE_FULL
