"""Cosines and sines of the forms with norms and 8-bit caches, at most 2^-23 off.

The fp32 gradient of a norm's weights is g x r: of one token of ones (r = 1) whose gradient is 1 in the first
element of a pair and 0 in the second, it is the pair's cosine and minus its sine, to the last bit.  With
base 1 and an axis for each pair, a position p turns its pair by p t 2^-64 turns (t the table's number), of
which the nearest multiple of 2^-32 counts: p = f 2^32 / t modulo 2^64 gives any of those, f."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib

DEV = torch.device("cuda", 0)


def cosines_and_sines(rope, f, D, pairing):
    """Of pair i at f[i] * 2^-32 turns."""
    n = D // 2
    turn = _lib.host().table_turns(rope._table)[0][0]
    even = (turn & -turn).bit_length() - 1
    inverse = pow(turn >> even, -1, 1 << 64)
    p = [((int(x) << 32 >> even) * inverse) % (1 << 64) for x in f]
    assert all((a * turn + 0x80000000) >> 32 & 0xFFFFFFFF == int(x) for a, x in zip(p, f))
    pos = torch.tensor(np.array(p, dtype=np.uint64).view(np.int64), device=DEV).view(n, 1, 1)
    x = torch.ones(1, 1, 1, D, dtype=torch.bfloat16, device=DEV)
    dy = torch.zeros_like(x)
    first = slice(0, n) if pairing == "half" else slice(0, D, 2)
    second = slice(n, D) if pairing == "half" else slice(1, D, 2)
    dy[..., first] = 1
    w = torch.ones(D, device=DEV, requires_grad=True)
    y, _ = rope(x, x, pos, query_norm=w, key_norm=w.detach(), eps=1e-20)
    dw, = torch.autograd.grad(y, w, dy)
    return dw[first], -dw[second]


@pytest.mark.gpu
@pytest.mark.parametrize("D,pairing", [(256, "half"), (256, "adjacent"), (246, "half")])
def test_cosines_and_sines(D, pairing):
    n = D // 2
    rope = api.MultiAxisRotary(D, (1,) * n, base=1.0, pairing=pairing)
    rng = np.random.default_rng(D)
    near = np.arange(-40, 41)[None] + (np.arange(16) << 28)[:, None]  # quarters, and what lies farthest from them
    few = np.outer(1 << np.arange(32), np.array([1, -1])) + (np.arange(4) << 30)[:, None, None]
    f = np.concatenate([near.ravel(), few.ravel(), rng.integers(0, 1 << 32, 60000)]) % (1 << 32)
    f = np.concatenate([f, np.zeros(-len(f) % n, dtype=f.dtype)]).reshape(-1, n)
    got = [cosines_and_sines(rope, row, D, pairing) for row in f]
    c, s = (torch.stack([g[i] for g in got]).double().cpu().numpy() for i in range(2))
    phi = 2 * np.pi * (f.astype(np.int64) - ((f >> 31) << 32)) / 2.0 ** 32
    assert np.abs(c - np.cos(phi)).max() <= 2.0 ** -23 and np.abs(s - np.sin(phi)).max() <= 2.0 ** -23
    # Whole quarters are exact.
    q = f % (1 << 30) == 0
    assert np.array_equal(c[q], np.round(np.cos(phi[q]))) and np.array_equal(s[q], np.round(np.sin(phi[q])))
