"""CPU: appending refuses 8-bit caches and scales that share memory with one another (blocks of threads
would write over one another's), and takes those that merely lie within one another."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api

E4M3 = torch.float8_e4m3fn
B, H, T, C, D = 2, 2, 3, 70, 64
POS = torch.zeros(1, 2, 3, dtype=torch.int64)


def append(kc, vc, ks, vs):
    x = torch.zeros(B, T, H, D, dtype=torch.bfloat16)
    return api.MultiAxisRotary(D, (D // 2,)).append(x, x, x, POS, kc, vc, torch.zeros(B, dtype=torch.int32), key_scale=ks,
                                                    value_scale=vs, layout="bshd")


def cache():
    return torch.zeros(B, C, H, D, dtype=torch.uint8).view(E4M3)


def scale():
    return torch.ones(B, H, 2)


@pytest.mark.parametrize("shift", [16, D, H * D, C * H * D, -16])
def test_caches_that_overlap_are_refused(shift):
    store = torch.zeros(2 * B * C * H * D + 64, dtype=torch.uint8)
    one, other = (store[a:a + B * C * H * D].view(B, C, H, D).view(E4M3) for a in (max(-shift, 0), max(shift, 0)))
    with pytest.raises(ValueError, match="of their own"):
        append(one, other, scale(), scale())


def test_a_cache_over_every_other_slot_of_the_other_is_refused():
    store = torch.zeros(B, 2 * C, H, D, dtype=torch.uint8).view(E4M3)
    with pytest.raises(ValueError, match="of their own"):
        append(store[:, :C], store.view(torch.uint8)[:, ::2].view(E4M3), scale(), scale())


@pytest.mark.parametrize("shift", [1, 2])
def test_scales_that_overlap_are_refused(shift):
    store = torch.ones(B * H * 2 + 2)
    one, other = (store[a:a + B * H * 2].view(B, H, 2) for a in (0, shift))
    with pytest.raises(ValueError, match="of their own"):
        append(cache(), cache(), one, other)


def test_scales_within_a_cache_are_refused():
    store = torch.zeros(B * C * H * D, dtype=torch.uint8)
    with pytest.raises(ValueError, match="of their own"):
        append(store.view(B, C, H, D).view(E4M3), cache(), store[:4 * B * H * 2].view(torch.float32).view(B, H, 2), scale())


def test_caches_and_scales_beside_one_another_are_taken():
    """Refused only for want of a GPU."""
    both = torch.zeros(B, C, 2, H, D, dtype=torch.uint8).view(E4M3)
    in_heads = torch.zeros(B, C, H, 2, D, dtype=torch.uint8).view(E4M3)
    scales = torch.ones(B, H, 2, 2)
    for kc, vc, ks, vs in ((both[:, :, 0], both[:, :, 1], scales[:, :, 0], scales[:, :, 1]),
                           (in_heads[..., 0, :], in_heads[..., 1, :], scale(), scale())):
        with pytest.raises(RuntimeError, match="CUDA"):
            append(kc, vc, ks, vs)
