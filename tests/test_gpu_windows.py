"""Queries and keys that are windows of one another: tokens whose rows overlap in memory, as
``unfold`` makes them, where a new tensor of the same stride order would not have its rows whole."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api

DEV = torch.device("cuda", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("step", [1, 3, 8])
@pytest.mark.parametrize("D,T", [(64, 9), (16, 40)])
def test_windows_give_the_same_bits_as_their_copies(layout, step, D, T):
    g = torch.Generator().manual_seed(D + step)
    base = torch.randn(2, 3, (T - 1) * step + D, generator=g).bfloat16().to(DEV)
    q = base.unfold(2, D, step)  # [2, 3, T, D], stride `step` from token to token
    k = base[:, :1].unfold(2, D, step)
    if layout == "bshd":
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    rope = api.MultiAxisRotary(D, (D // 4, D // 4))
    pos = torch.randint(0, 999, (2, 2, T), generator=g).to(DEV)
    want = rope(q.contiguous(), k.contiguous(), pos, layout=layout)
    got = rope(q, k, pos, layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    yq, yk = rope(x, y, pos, layout=layout)
    gq, gk = torch.autograd.grad((yq, yk), (x, y), (q, k))
    hq, hk = torch.autograd.grad(rope(x, y, pos, layout=layout), (x, y), (q.contiguous(), k.contiguous()))
    assert torch.equal(gq, hq) and torch.equal(gk, hk)

    def appended(q, k):
        shape = (2, 1, T, D) if layout == "bhsd" else (2, T, 1, D)
        cache = [torch.zeros(shape, dtype=q.dtype, device=DEV) for _ in range(2)]
        n = torch.zeros(2, dtype=torch.int32, device=DEV)
        return [*rope.append(q, k, k, pos, *cache, n, layout=layout), *cache]

    assert all(torch.equal(a, b) for a, b in zip(appended(q, k), appended(q.contiguous(), k.contiguous()), strict=True))
    if D == 64:
        prefix = torch.randn((1, 30, D) if layout == "bhsd" else (30, 1, D), generator=g).bfloat16().to(DEV)
        n = torch.full((2,), T, dtype=torch.int32, device=DEV)
        call = lambda q, k: api.shared_prefix_attention(q, prefix, prefix, k, k, n, layout=layout)  # noqa: E731
        assert torch.equal(call(q, k), call(q.contiguous(), k.contiguous()))
