"""The decode example: every step agrees with plain torch, across evictions."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT
from fa2_with_4d_mask_b200 import _lib


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(batch=3, steps=130), dict(batch=20, steps=50, heads=8, kv_heads=8, head_dim=64, capacity=40, keep=30, recent=10)])
def test_decode_example(kw):
    spec = importlib.util.spec_from_file_location("shared_prefix_decode", ROOT / "examples" / "shared_prefix_decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    seen = []

    def observe(step, *rest):
        example.compare(step, *rest)
        seen.append(step)

    x, lengths, _ = example.decode(observe=observe, **kw)
    assert len(seen) == kw["steps"] and bool(torch.isfinite(x).all())
    capacity, keep = kw.get("capacity", 96), kw.get("keep", 64)
    extra = (kw["steps"] - capacity - 1) % (capacity - keep) + 1
    assert lengths.tolist() == [keep + extra] * kw["batch"]
    again, _, _ = example.decode(**kw)
    assert torch.equal(again, x)
    assert _lib.device_status(torch.device("cuda", 0)) == 0
