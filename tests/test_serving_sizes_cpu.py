"""CPU: caches without a head or without elements are refused, not answered with lengths that
nothing has written."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api


@pytest.mark.parametrize("H,D", [(0, 64), (2, 0), (0, 0)])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_evict_needs_a_head_and_an_element(H, D, layout):
    shape = (2, H, 8, D) if layout == "bhsd" else (2, 8, H, D)
    cache, n = torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="at least one head"):
        api.evict_by_weight(cache, cache, torch.zeros(2, H, 8), n, keep=4, layout=layout)
