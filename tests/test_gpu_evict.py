"""Eviction by weight: the kept slots and everything copied are equal to the plain form's."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from oracle.serving import evict_ref

DEV = torch.device("cuda", 0)


def cache(g, B, Hk, C, D, dtype, layout):
    return torch.randn((B, Hk, C, D) if layout == "bhsd" else (B, C, Hk, D), generator=g).to(dtype).to(DEV)


def check(k, v, w, lengths, keep, sinks, recent, layout, got):
    ko, vo, wo, new, index = got
    B, Hk, C = w.shape
    n = lengths.clamp(0, C)
    ref = evict_ref(w, lengths, keep, sinks, recent)
    assert torch.equal(index.cpu().long(), ref)
    assert torch.equal(new, n.clamp(max=keep).int())
    rows = [x if layout == "bhsd" else x.transpose(1, 2) for x in (k, v, ko, vo)]
    for b in range(B):
        for h in range(Hk):
            m = int(new[b])
            at = ref[b, h, :m].to(DEV)
            for src, dst in ((rows[0], rows[2]), (rows[1], rows[3])):
                assert torch.equal(dst[b, h, :m].view(torch.int16), src[b, h, at].view(torch.int16))
                assert not dst[b, h, m:keep].any()
            assert torch.equal(wo[b, h, :m].view(torch.int32), w[b, h, at].view(torch.int32)) and not wo[b, h, m:keep].any()


CASES = [
    # (B, Hk, C, D, keep, sinks, recent, dtype, layout)
    (1, 1, 1, 64, 1, 0, 0, torch.bfloat16, "bhsd"),
    (1, 1, 2, 8, 1, 0, 1, torch.bfloat16, "bshd"),
    (2, 3, 37, 96, 20, 4, 7, torch.float16, "bshd"),
    (3, 2, 700, 64, 512, 4, 64, torch.bfloat16, "bhsd"),
    (1, 8, 1031, 128, 500, 0, 0, torch.bfloat16, "bshd"),
    (2, 2, 5000, 128, 1234, 1, 1233, torch.float16, "bhsd"),  # no room for the middle
    (70, 8, 300, 64, 200, 2, 50, torch.bfloat16, "bshd"),  # one CTA a head
    (1, 2, 20011, 256, 9000, 4, 1000, torch.bfloat16, "bhsd"),
    (1, 1, 140003, 16, 70000, 4, 999, torch.float16, "bhsd"),  # a slice is more than a CTA keeps
    (1, 2, 8193, 64, 8192, 0, 0, torch.bfloat16, "bshd"),
    (2, 2, 400, 20, 300, 3, 30, torch.float16, "bhsd"),  # rows that are no multiple of 16 bytes
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hk,C,D,keep,sinks,recent,dtype,layout", CASES)
def test_keeps_the_heaviest(B, Hk, C, D, keep, sinks, recent, dtype, layout):
    g = torch.Generator().manual_seed(C)
    k, v = (cache(g, B, Hk, C, D, dtype, layout) for _ in range(2))
    w = torch.randn(B, Hk, C, generator=g).mul(3).exp().to(DEV)
    lengths = torch.randint(0, C + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
    lengths[0] = C
    got = api.evict_by_weight(k, v, w, lengths, keep=keep, sinks=sinks, recent=recent, layout=layout)
    check(k, v, w, lengths, keep, sinks, recent, layout, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zeros", "few values", "signed zeros", "nan and inf", "subnormal", "negative"])
@pytest.mark.parametrize("C", [600, 9001])
def test_ties_and_special_weights(kind, C):
    g = torch.Generator().manual_seed(7)
    w = torch.zeros(2, 2, C)
    if kind == "few values":
        w = torch.randint(0, 3, (2, 2, C), generator=g).float()
    elif kind == "signed zeros":
        w = torch.where(torch.rand(2, 2, C, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "nan and inf":
        r = torch.rand(2, 2, C, generator=g)
        w = torch.where(r < 0.3, float("nan"), torch.where(r < 0.4, float("inf"), torch.where(r < 0.6, -float("inf"), r)))
    elif kind == "subnormal":
        w = torch.randint(0, 9, (2, 2, C), generator=g).float() * 1.4e-45
    elif kind == "negative":
        w = torch.randn(2, 2, C, generator=g)
    w = w.to(DEV)
    k, v = (cache(g, 2, 2, C, 64, torch.bfloat16, "bhsd") for _ in range(2))
    lengths = torch.tensor([C, C - 77], dtype=torch.int32, device=DEV)
    for keep, sinks, recent in ((C // 2, 4, 64), (C - 80, 0, 0), (3, 1, 1)):
        got = api.evict_by_weight(k, v, w, lengths, keep=keep, sinks=sinks, recent=recent)
        check(k, v, w, lengths, keep, sinks, recent, "bhsd", got)


@pytest.mark.gpu
def test_stale_slots_are_not_read_and_lengths_are_clamped():
    g = torch.Generator().manual_seed(1)
    k, v = (cache(g, 4, 2, 200, 64, torch.float16, "bshd") for _ in range(2))
    w = torch.rand(4, 2, 200, generator=g).to(DEV)
    lengths = torch.tensor([150, 0, -3, 999], dtype=torch.int32, device=DEV)
    for x in (k, v):
        x[0, 150:], x[1], x[2] = float("nan"), float("nan"), float("nan")
    w[0, :, 150:], w[1:3] = float("inf"), float("inf")
    got = api.evict_by_weight(k, v, w, lengths, keep=100, sinks=2, recent=10, layout="bshd")
    check(k, v, w, lengths, 100, 2, 10, "bshd", got)
    assert got[3].tolist() == [100, 0, 0, 100] and bool(torch.isfinite(got[0]).all())


@pytest.mark.gpu
def test_strides_and_out():
    """Caches and weights as views, an output with more slots than are kept."""
    g = torch.Generator().manual_seed(2)
    k = cache(g, 2, 3, 90, 80, torch.bfloat16, "bhsd")[..., 8:72]
    v = cache(g, 2, 3, 90, 64, torch.bfloat16, "bshd").transpose(1, 2)
    w = torch.rand(2, 3, 130, generator=g).to(DEV)[..., 7:97]
    lengths = torch.tensor([90, 61], dtype=torch.int32, device=DEV)
    out = (torch.full((2, 3, 75, 64), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((2, 75, 3, 64), 7.0, dtype=torch.bfloat16, device=DEV).transpose(1, 2),
           torch.full((2, 3, 75), 7.0, device=DEV))
    got = api.evict_by_weight(k, v, w, lengths, keep=60, sinks=1, recent=9, out=out)
    assert got[0] is out[0] and got[1] is out[1] and got[2] is out[2]
    check(k, v, w, lengths, 60, 1, 9, "bhsd", got)
    assert all(bool((x[:, :, 60:] == 7).all()) for x in out)
    with pytest.raises(ValueError, match="share memory"):
        api.evict_by_weight(k, v, w, lengths, keep=60, out=(k, torch.empty_like(v), torch.empty_like(w)))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    store = torch.empty(2 ** 31 + 65536, dtype=torch.bfloat16, device=DEV)
    k = store.as_strided((2, 1, 200, 64), (2 ** 31 + 8, 64 * 200, 64, 1))
    g = torch.Generator().manual_seed(0)
    k.copy_(cache(g, 2, 1, 200, 64, torch.bfloat16, "bhsd"))
    w = torch.rand(2, 1, 200, generator=g).to(DEV)
    lengths = torch.tensor([200, 200], dtype=torch.int32, device=DEV)
    check(k, k, w, lengths, 99, 0, 5, "bhsd", api.evict_by_weight(k, k, w, lengths, keep=99, recent=5))
