"""Norms with the rotary turn where every thread takes many rows: the feed's ring goes round, ranges of
several heads with what is left of them, grids of more blocks than run at once; prompts whose queries
share a block.  Bounds are those of ``test_gpu_norm_rotary`` and ``test_gpu_cache8``, but for the weights'
gradients: sums of N rows run in chains (a thread's rows, a block's threads, the blocks by 32
threads, those), below 400 additions for these sizes, so their rounding is at most 400 * 2^-24 of
sum G |xh|."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import norm_rotary_grads
from test_gpu_cache8 import check_append
from test_gpu_norm_rotary import DEV, U, close, forward_close

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def gradients_close(dx, dw, x, w, dy, pos, sections, eps, **kw):
    _, rx, rw = norm_rotary_grads(x, w, dy, pos, sections, eps=eps, **kw)
    x, w, D = x.double(), w.double(), x.shape[-1]
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    xh, G = x * r, dy.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
    f = 2 * (D + 64) * 2.0 ** -24 + 2.0 ** -19
    size = r * G * (w.abs().max() + xh.abs() * (w * xh).abs().mean(-1, keepdim=True))
    close(dx, rx, U[dx.dtype] * rx.abs() + f * size + 2.0 ** -25)
    close(dw, rw, U[dw.dtype] * rw.abs() + (f + 400 * 2.0 ** -24) * (G * xh.abs()).sum((0, 1, 2)) + 2.0 ** -25)


CASES = [
    # (B, T, Hq, Hk, D, rotary_dim, sections, pairing, dtype, weight dtype, layout)
    (1, 8192, 32, 8, 128, None, (16, 24, 24), "half", BF16, F32, "bshd"),
    (2, 16500, 16, 8, 256, None, (128,), "half", FP16, FP16, "bshd"),  # three and two grids' worth of blocks
    (1, 20001, 18, 5, 64, None, (8, 24), "adjacent", BF16, BF16, "bhsd"),  # ranges of 9 heads
    (1, 9001, 37, 3, 96, 64, (32,), "half", FP16, F32, "bshd"),  # 13, 13 and 11
    (1, 5000, 7, 3, 80, 36, (9, 9), "half", BF16, F32, "bhsd"),  # pair by pair
]


def inputs(B, T, Hq, Hk, D, rot, sections, pairing, dtype, wide, layout):
    g = torch.Generator(DEV).manual_seed(T + D)
    rope = api.MultiAxisRotary(D, sections, base=1e4, rotary_dim=rot, pairing=pairing)
    shape = lambda H: (B, H, T, D) if layout == "bhsd" else (B, T, H, D)  # noqa: E731
    q, k, dq, dk = ((torch.randn(shape(H), generator=g, device=DEV) * f).to(dtype) for H, f in ((Hq, 2.0), (Hk, 0.3), (Hq, 1.0), (Hk, 1.0)))
    pos = torch.randint(-50, 100000, (len(sections), B, T), generator=g, device=DEV, dtype=torch.int32)
    w = [(1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(wide) for _ in range(2)]
    return rope, q, k, dq, dk, pos, w, dict(base=1e4, rotary_dim=rot, pairing=pairing, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients_over_many_rows(case):
    sections, layout, eps = case[6], case[10], 1e-5
    rope, q, k, dq, dk, pos, (wq, wk), kw = inputs(*case)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    yq, yk = rope(q, k, pos, query_norm=wq, key_norm=wk, eps=eps, layout=layout)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk), retain_graph=True)
    for y, x, d, gx, w, gw in ((yq, q, dq, grads[0], wq, grads[2]), (yk, k, dk, grads[1], wk, grads[3])):
        forward_close(y.detach(), x.detach(), w.detach(), pos, sections, eps, **kw)
        gradients_close(gx, gw, x.detach(), w.detach(), d, pos, sections, eps, **kw)
    again = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("Hq,Hk,D,rot,sections,normed", [(9, 2, 128, None, (64,), True), (6, 3, 64, None, (8, 24), True),
                                                         (32, 2, 96, 32, (16,), False), (9, 1, 80, 36, (18,), True)])
def test_prompts_into_8_bit_caches_whose_queries_share_blocks(Hq, Hk, D, rot, sections, normed, code):
    """Blocks of 8, 4 and 16 query heads, with one, two and none left over."""
    rope, q, k, _, _, pos, w, kw = inputs(2, 4300, Hq, Hk, D, rot, sections, "half", BF16, F32, "bshd")
    v = torch.randn(k.shape, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(BF16)
    kc, vc = (torch.zeros(2, 4400, Hk, D, dtype=torch.uint8, device=DEV).view(code) for _ in range(2))
    ks, vs = (torch.ones(2, Hk, 69, device=DEV) for _ in range(2))
    lengths = torch.tensor([0, 37], dtype=torch.int32, device=DEV)
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, lengths, sections, "bshd", weights=w if normed else None, base=1e4,
                 rotary_dim=rot)
    if normed:  # again: the queries against the formula (the slots' scales are there already)
        got, _ = rope.append(q, k, v, pos, kc, vc, lengths, query_norm=w[0], key_norm=w[1], key_scale=ks, value_scale=vs, layout="bshd")
        forward_close(got, q, w[0], pos, sections, 1e-6, **kw)
    assert _lib.device_status(DEV) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk,D,rot", [(9, 9, 128, None), (32, 6, 64, 32), (18, 9, 80, 36)])
def test_prompts_into_16_bit_caches_whose_heads_share_blocks(Hq, Hk, D, rot):
    sections = ((D if rot is None else rot) // 2,)
    rope, q, k, _, _, pos, w, kw = inputs(2, 4300, Hq, Hk, D, rot, sections, "half", BF16, F32, "bshd")
    v = torch.randn(k.shape, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(BF16)
    kc, vc = (torch.zeros(2, 4400, Hk, D, dtype=BF16, device=DEV) for _ in range(2))
    lengths = torch.tensor([0, 37], dtype=torch.int32, device=DEV)
    got, new = rope.append(q, k, v, pos, kc, vc, lengths, query_norm=w[0], key_norm=w[1], layout="bshd")
    forward_close(got, q, w[0], pos, sections, 1e-6, **kw)
    for b, n in enumerate(lengths.tolist()):
        forward_close(kc[b:b + 1, n:n + 4300], k[b:b + 1], w[1], pos[:, b:b + 1], sections, 1e-6, **kw)
        assert torch.equal(vc[b, n:n + 4300], v[b])
        assert not kc[b, :n].any() and not kc[b, n + 4300:].any() and not vc[b, :n].any() and not vc[b, n + 4300:].any()
    assert new.tolist() == [4300, 4337] and _lib.device_status(DEV) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradients_of_inputs_that_are_broadcast(dtype):
    """One head of one request for all of them, through strides of 0: the kernels read the same rows as
    of a copy, so the weights' gradients are the same bits, and the input's is the sum of the
    copy's, added in 32 bits (8 terms) and rounded once."""
    g = torch.Generator(DEV).manual_seed(5)
    rope = api.MultiAxisRotary(64, (8, 12, 12))
    pos = torch.randint(0, 5000, (3, 2, 9), generator=g, device=DEV)
    one = torch.randn(1, 1, 9, 64, generator=g, device=DEV).to(dtype).requires_grad_()
    k, dy = (torch.randn(2, H, 9, 64, generator=g, device=DEV).to(dtype) for H in (2, 4))
    w, v = (torch.linspace(0.5, 1.5, 64, device=DEV).requires_grad_() for _ in range(2))
    full = one.detach().expand(2, 4, -1, -1).contiguous().requires_grad_()
    d1, dw = torch.autograd.grad(rope(one.expand(2, 4, -1, -1), k, pos, query_norm=w, key_norm=w)[0], (one, w), dy)
    d2, dv = torch.autograd.grad(rope(full, k, pos, query_norm=v, key_norm=v)[0], (full, v), dy)
    assert torch.equal(dw, dv)
    d2 = d2.double()
    want, size = d2.sum((0, 1), keepdim=True), d2.abs().sum((0, 1), keepdim=True)
    close(d1, want, U[dtype] * want.abs() + 8 * 2.0 ** -24 * size + 2.0 ** -25)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 22])
def test_gradients_where_squares_leave_32_bits(D):
    """Rows of zeros beside the least epsilon, whose r^2 is beyond fp32: dx = r w g.  Rows whose squares are
    infinite in 32 bits are normalised to zeros whatever they hold, so their gradient is 0."""
    rope = api.MultiAxisRotary(D, (D // 2,))
    x = torch.ones(1, 1, 4, D, dtype=BF16, device=DEV)
    x[0, 0, 1] = 0
    x[0, 0, 2] = 3e38
    x[0, 0, 3] = 2.0 ** -100
    w = torch.linspace(0.5, 1.5, D, device=DEV)
    pos = torch.zeros(1, 1, 4, dtype=torch.int64, device=DEV)
    dy = torch.ones_like(x)
    dy[..., ::2] = 0.5
    eps = 2.0 ** -130
    leaf, v = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = rope(leaf, x, pos, query_norm=v, key_norm=v, eps=eps)
    assert not y[0, 0, 1:3].any()
    dx, dw = torch.autograd.grad(y, (leaf, v), dy)
    rows = [0, 1, 3]
    gradients_close(dx[:, :, rows], dw, x[:, :, rows], w, dy[:, :, rows], pos[..., rows], (D // 2,), eps, base=1e4)
    assert not dx[0, 0, 2].any()
