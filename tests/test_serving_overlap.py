"""Which outputs of evict_by_weight share memory with its inputs, or with each other, is
decided by their elements, not by the spans from their first to their last."""

from __future__ import annotations

import itertools

import pytest
import torch

import tilelang_fa2_4d_mask as api

B, C, H, D, KEEP = 2, 6, 3, 8, 4


def evict(k, v, out_k, out_v, w=None, out_w=None, lengths=None, layout="bshd"):
    slots = 1 if layout == "bshd" else 2
    w = torch.zeros(B, H, k.shape[slots]) if w is None else w
    out_w = torch.zeros(B, H, out_k.shape[slots]) if out_w is None else out_w
    n = torch.zeros(B, dtype=torch.int32) if lengths is None else lengths
    return api.evict_by_weight(k, v, w, n, keep=KEEP, out=(out_k, out_v, out_w), layout=layout)


def accepted(*args, **kw):
    with pytest.raises(RuntimeError, match="CUDA"):  # as far as the device
        evict(*args, **kw)


def refused(*args, **kw):
    with pytest.raises(ValueError, match="share memory"):
        evict(*args, **kw)


def new(slots):
    return torch.zeros(B, slots, H, D, dtype=torch.bfloat16)


def test_keys_and_values_in_one_tensor():
    for dim, shape in ((2, (B, C, 2, H, D)), (3, (B, C, H, 2, D)), (1, (B, 2, C, H, D)), (0, (2, B, C, H, D))):
        out = torch.zeros(shape, dtype=torch.bfloat16)
        accepted(new(C), new(C), out.select(dim, 0), out.select(dim, 1))
        refused(new(C), new(C), out.select(dim, 0), out.select(dim, 0))
    both = torch.zeros(B, C, H, 2 * D, dtype=torch.bfloat16)
    accepted(new(C), new(C), both[..., :D], both[..., D:])
    refused(new(C), new(C), both[..., :D], both[..., D // 2 : D // 2 + D])


def test_two_sets_of_caches_cut_from_one_pool():
    pool = torch.zeros(B, 4, C, H, D, dtype=torch.bfloat16)
    accepted(pool[:, 0], pool[:, 1], pool[:, 2], pool[:, 3])
    refused(pool[:, 0], pool[:, 1], pool[:, 1], pool[:, 3])
    refused(pool[:, 0], pool[:, 1], pool[:, 2], pool[:, 0])
    # Slots of the pool in turn; halves of the requests' slots.
    turns = torch.zeros(B, 2 * C, H, D, dtype=torch.bfloat16)
    accepted(turns[:, 0::2], new(C), turns[:, 1::2], new(C))
    accepted(turns[:, :C], new(C), turns[:, C:], new(C))
    refused(turns[:, 0::2], new(C), turns[:, 2:8], new(C))
    refused(turns[:, :C], new(C), turns[:, C - 1 : 2 * C - 1], new(C))
    # Heads of the pool in turn, in the other layout.
    heads = torch.zeros(B, 2 * H, C, D, dtype=torch.bfloat16)
    k = torch.zeros(B, H, C, D, dtype=torch.bfloat16)
    accepted(heads[:, 0::2], k, heads[:, 1::2], k.clone(), layout="bhsd")
    refused(heads[:, :H], k, heads[:, H - 1 : 2 * H - 1], k.clone(), layout="bhsd")


def test_weights_and_lengths_beside_the_caches():
    """Elements of 4 bytes beside elements of 2."""
    buffer = torch.zeros(B, H, 2 * C)
    accepted(new(C), new(C), new(KEEP), new(KEEP), w=buffer[..., :C], out_w=buffer[..., C : C + KEEP])
    refused(new(C), new(C), new(KEEP), new(KEEP), w=buffer[..., :C], out_w=buffer[..., C - 1 : C - 1 + KEEP])
    size = B * KEEP * H * D
    pool = torch.zeros(size + 2 * B, dtype=torch.bfloat16)
    out = pool[:size].view(B, KEEP, H, D)
    accepted(new(C), new(C), out, new(KEEP), lengths=pool[size:].view(torch.int32))
    refused(new(C), new(C), out, new(KEEP), lengths=pool[size - 2 : size + 2 * B - 2].view(torch.int32))


def test_outputs_may_not_share_with_each_other():
    pool = torch.zeros(B * KEEP * H * D, dtype=torch.bfloat16)
    k = pool.view(B, KEEP, H, D)
    refused(new(C), new(C), k, new(KEEP), out_w=pool[: B * H * KEEP * 2].view(torch.float32).view(B, H, KEEP))
    refused(new(C), new(C), new(KEEP), k, out_w=pool[: B * H * KEEP * 2].view(torch.float32).view(B, H, KEEP))


def test_against_the_elements_themselves():
    """Views of one buffer with many strides: refused exactly where an element is shared."""
    g = torch.Generator().manual_seed(0)
    found = {True: 0, False: 0}
    for _ in range(400):
        pool = torch.zeros(1 << 14, dtype=torch.bfloat16)
        views = []
        for slots in (C, KEEP):
            dims = [B, slots, H]
            strides = [0, 0, 0]
            step = D + int(torch.randint(0, 3, (), generator=g)) * D
            for i in torch.randperm(3, generator=g).tolist():
                strides[i] = step
                step *= dims[i] + int(torch.randint(0, 2, (), generator=g))
            at = int(torch.randint(0, 1500, (), generator=g))
            views.append(pool.as_strided((B, slots, H, D), (*strides, 1), at))
        elements = [{x.storage_offset() + sum(i * s for i, s in zip(at, x.stride())) + d
                     for at in itertools.product(*map(range, x.shape[:3])) for d in range(D)} for x in views]
        shared = bool(elements[0] & elements[1])
        found[shared] += 1
        (refused if shared else accepted)(views[0], new(C), views[1], new(KEEP))
    assert min(found.values()) > 30


@pytest.mark.gpu
def test_an_interleaved_output_is_written():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).bfloat16().cuda()  # noqa: E731
    k, v, w = r(B, 40, H, 64), r(B, 40, H, 64), torch.rand(B, H, 40, generator=g).cuda()
    n = torch.tensor([40, 33], dtype=torch.int32, device="cuda")
    want = api.evict_by_weight(k, v, w, n, keep=20, sinks=2, recent=5, layout="bshd")
    out = torch.zeros(B, 20, 2, H, 64, dtype=torch.bfloat16, device="cuda")
    got = api.evict_by_weight(k, v, w, n, keep=20, sinks=2, recent=5, layout="bshd",
                              out=(out[:, :, 0], out[:, :, 1], torch.zeros(B, H, 20, device="cuda")))
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
