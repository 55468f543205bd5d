"""The rotary's 16-byte path and its path of single elements round alike: where rows lie in memory
changes no bit of the result, over enough elements that a fused multiply-add in another place shows
(about one in 50000 bf16 results then differs)."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api

DEV = torch.device("cuda", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_rows_past_a_16_byte_boundary_give_the_same_bits(dtype, pairing):
    g = torch.Generator().manual_seed(1)
    B, H, T, D = 2, 8, 700, 128
    rope = api.MultiAxisRotary(D, (16, 24, 24), pairing=pairing)
    pos = torch.randint(0, 5000, (3, B, T), generator=g).to(DEV)
    q, dq = (torch.randn(B, H, T, D, generator=g).to(dtype).to(DEV) for _ in range(2))

    def shifted(x):
        return torch.empty(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape).copy_(x)

    def both(x, dx):
        x = x.detach().requires_grad_()
        y, _ = rope(x, x.detach()[:, :1], pos)
        return y, *torch.autograd.grad(y, x, dx)

    def appended(x):
        cache = [torch.zeros(B, H, T, D, dtype=dtype, device=DEV) for _ in range(2)]
        y, _ = rope.append(x, x, x, pos, *cache, torch.zeros(B, dtype=torch.int32, device=DEV))
        return y, cache[0]

    assert all(torch.equal(a, b) for a, b in zip(both(q, dq), both(shifted(q), shifted(dq)), strict=True))
    assert all(torch.equal(a, b) for a, b in zip(appended(q), appended(shifted(q)), strict=True))
    assert torch.equal(appended(q)[0], both(q, dq)[0])
