"""Caches and weights written in place are written as by an in-place operation of torch: refused
where they require a gradient, and seen by autograd where their old values were saved."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api

B, H, T, D, C = 2, 2, 3, 64, 8


def new(dev, slots=T):
    return torch.zeros(B, H, slots, D, dtype=torch.bfloat16, device=dev)


def calls(dev):
    """name -> (written tensors, call)."""
    n = torch.full((B,), 2, dtype=torch.int32, device=dev)
    pos = torch.zeros(1, B, T, dtype=torch.int64, device=dev)
    rope = api.MultiAxisRotary(D, (D // 2,))
    w = lambda: torch.zeros(B, H, C, device=dev)  # noqa: E731
    return {
        "append": ([new(dev, C), new(dev, C), w()],
                   lambda k, v, w: rope.append(new(dev), new(dev), new(dev), pos, k, v, n, weights=w)),
        "attend": ([w()], lambda w: api.shared_prefix_attention(new(dev), None, None, new(dev, C), new(dev, C), n, weights=w)),
        "evict": ([new(dev, C), new(dev, C), w()],
                  lambda k, v, x: api.evict_by_weight(new(dev, C), new(dev, C), w(), n, keep=4, out=(k, v, x))),
    }


EACH = [(name, i) for name, (written, _) in calls("cpu").items() for i in range(len(written))]


@pytest.mark.parametrize("name,i", EACH)
def test_written_tensors_that_require_a_gradient_are_refused(name, i):
    written, call = calls("cpu")[name]
    written[i].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        call(*written)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # as torch allows it
        call(*written)


@pytest.mark.gpu
@pytest.mark.parametrize("name,i", EACH)
def test_autograd_sees_the_write(name, i):
    written, call = calls("cuda")[name]
    x = torch.ones_like(written[i], requires_grad=True)
    y = (x * written[i]).sum()  # saves written[i]
    before = written[i]._version
    call(*written)
    assert written[i]._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(calls("cpu")))
def test_inference_tensors_can_be_written(name):
    with torch.inference_mode():
        written, call = calls("cuda")[name]
        call(*written)
