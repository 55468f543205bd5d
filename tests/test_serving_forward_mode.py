"""Tensors with a forward-mode tangent are refused by the operators around the attention (as
the attention itself refuses them), not run without it."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import tilelang_fa2_4d_mask as api

B, H, T, D, C = 2, 2, 3, 64, 8
POS = torch.zeros(1, B, T, dtype=torch.int64)


def new(slots=T, shape=None):
    return torch.zeros(shape or (B, H, slots, D), dtype=torch.bfloat16)


def calls():
    n = torch.zeros(B, dtype=torch.int32)
    rope = api.MultiAxisRotary(D, (D // 2,))
    w = torch.zeros(B, H, C)
    return {
        "rotary": ([new(), new()], lambda q, k: rope(q, k, POS)),
        "append": ([new(), new(), new(), new(C), new(C), w],
                   lambda q, k, v, kc, vc, w: rope.append(q, k, v, POS, kc, vc, n, weights=w)),
        "attend": ([new(), new(shape=(H, 5, D)), new(shape=(H, 5, D)), new(C), new(C), w],
                   lambda q, pk, pv, k, v, w: api.shared_prefix_attention(q, pk, pv, k, v, n, weights=w)),
        "evict": ([new(C), new(C), w], lambda k, v, w: api.evict_by_weight(k, v, w, n, keep=4)),
    }


@pytest.mark.parametrize("name,i", [(name, i) for name, (tensors, _) in calls().items() for i in range(len(tensors))])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_tangent_is_refused(name, i, grad_mode):
    tensors, call = calls()[name]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        tensors[i] = forward_ad.make_dual(tensors[i], torch.ones_like(tensors[i]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*tensors)


@pytest.mark.parametrize("name", list(calls()))
def test_without_a_tangent_nothing_is_refused(name):
    tensors, call = calls()[name]
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="CUDA"):
        call(*tensors)
    dual = tensors[0]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(tensors[0], torch.ones_like(tensors[0]))
    with pytest.raises(RuntimeError, match="CUDA"):  # its level has ended
        call(dual, *tensors[1:])


@pytest.mark.gpu
def test_a_tangent_of_the_gradient_is_refused():
    """Forward over reverse: the tangent reaches the rotary in its backward."""
    x = torch.randn(1, 2, 4, D, device="cuda").bfloat16().requires_grad_()
    y, _ = api.MultiAxisRotary(D, (D // 2,))(x, x, torch.zeros(1, 1, 4, dtype=torch.int64, device="cuda"))
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="jvp|forward-mode"):
            torch.autograd.grad(y, x, dy)
