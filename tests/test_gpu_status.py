"""The device status word is shared by every operator of the library: a checked backward reports
its own kernels' bits and leaves the sign that a cache was full to who reads it."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib, fa2

DEV = torch.device("cuda", 0)


def fill_a_cache():
    x = torch.ones(1, 1, 3, 64, dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    api.MultiAxisRotary(64, (32,)).append(x, x, x, torch.zeros(1, 1, 3, dtype=torch.int64, device=DEV), cache, cache.clone(), n)


def train():
    q = torch.randn(1, 2, 130, 64, device=DEV).bfloat16().requires_grad_()
    api.tilelang_flash_attention(q, q, q, is_causal=True).sum().backward()
    return q.grad


@pytest.mark.gpu
def test_a_checked_backward_leaves_the_full_cache_to_its_reader(monkeypatch):
    monkeypatch.setattr(fa2, "_CHECK_STATUS", True)
    assert api.device_status(DEV) == 0
    fill_a_cache()
    assert bool(torch.isfinite(train()).all())
    assert api.device_status(DEV) == api.DEV_CACHE_FULL == _lib.DEV_CACHE_FULL
    assert api.device_status(DEV) == 0


@pytest.mark.gpu
def test_a_checked_backward_that_raises_tells_of_both(monkeypatch):
    monkeypatch.setattr(fa2, "_CHECK_STATUS", True)
    fill_a_cache()
    lib = _lib.load_library()
    assert lib.fa4d_check_wait_timeout(0, 1000, None) == 0  # sets its bit and returns
    with pytest.raises(RuntimeError, match=r"bounded wait \(device status 0x4\).*cache was full"):
        train()
    assert api.device_status(DEV) == 0
