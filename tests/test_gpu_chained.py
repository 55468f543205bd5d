"""The operators one behind the other on a stream, each reading what the one ahead has written,
without a kernel of another kind between them: the same bits as with a synchronisation after
every call."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib

DEV = torch.device("cuda", 0)


def rounds(n, B, T, Hq, Hk, D, P, C, keep, layout, settle):
    """n rounds of attend, evict, append and attend between two sets of caches; everything made
    beforehand.  The lengths that append returns are also the next positions."""
    g = torch.Generator().manual_seed(B + D)
    dt = torch.bfloat16

    def heads(H, S):
        return torch.randn((B, H, S, D) if layout == "bhsd" else (B, S, H, D), generator=g).to(dt).to(DEV)

    pk, pv = (torch.randn((Hk, P, D) if layout == "bhsd" else (P, Hk, D), generator=g).to(dt).to(DEV) for _ in range(2))
    cache, spare = [heads(Hk, C), heads(Hk, C), torch.rand(B, Hk, C, generator=g).to(DEV)], None
    spare = [torch.zeros_like(x) for x in cache]
    news = [[heads(H, T) for H in (Hq, Hk, Hk)] for _ in range(n)]
    q0 = heads(Hq, T)
    lengths = torch.full((B,), C, dtype=torch.int32, device=DEV)
    rope = api.MultiAxisRotary(D, (D // 2,))
    seen = []
    torch.cuda.synchronize()

    def after(*got):
        seen.extend(got)
        if settle:
            torch.cuda.synchronize()

    q = q0
    for new in news:
        o = api.shared_prefix_attention(q, pk, pv, cache[0], cache[1], lengths, weights=cache[2], layout=layout)
        after(o)
        *spare, lengths, index = api.evict_by_weight(*cache, lengths, keep=keep, sinks=1, recent=T, out=tuple(spare), layout=layout)
        after(lengths, index)
        cache, spare = spare, cache
        at = lengths.view(1, B, 1).expand(1, B, T)
        q, lengths = rope.append(*new, at, cache[0], cache[1], lengths, weights=cache[2], layout=layout)
        after(q, lengths)
    torch.cuda.synchronize()
    return seen + cache


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C,keep,layout", [
    (1, 1, 8, 2, 128, 40, 300, 250, "bshd"),
    (3, 2, 4, 4, 64, 0, 90, 70, "bhsd"),
    (40, 1, 8, 2, 128, 2000, 200, 150, "bshd"),
    (16, 3, 8, 2, 256, 2100, 120, 100, "bhsd"),
    (2, 1, 4, 2, 64, 10, 9000, 8500, "bshd"),
])
def test_every_operator_sees_what_the_one_ahead_wrote(B, T, Hq, Hk, D, P, C, keep, layout):
    n = 40
    want = rounds(n, B, T, Hq, Hk, D, P, C, keep, layout, True)
    for _ in range(3):
        got = rounds(n, B, T, Hq, Hk, D, P, C, keep, layout, False)
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert _lib.device_status(DEV) == 0
