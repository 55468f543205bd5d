"""Attention over a shared prefix and own caches against the 64-bit formula.

Bound of the output: P is rounded to 16 bits before the product with V (u p |v| for each key),
the result once more (u |o|), and the logits carry the error of a 32-bit dot product of D
terms, at most e = (D + 8) 2^-24 max sum|q k| |scale| plus the exponential's 2^-21, twice
(numerator and denominator): |o - o64| <= u |o64| + (u + 2 e + 2^-20) sum p |v| + 2^-24,
u = 2^-8 (bf16) or 2^-11 (fp16).  Weights, in 32 bits: (2 e + 2^-19) of themselves, from
whatever was added to 2^-23 of it."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.serving import shared_prefix_ref

DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(g, B, T, Hq, Hk, D, P, C, dtype, layout):
    r = lambda *s: torch.randn(s, generator=g).to(dtype).to(DEV)  # noqa: E731
    if layout == "bhsd":
        return r(B, Hq, T, D), (r(Hk, P, D) if P else None), (r(Hk, P, D) if P else None), r(B, Hk, C, D), r(B, Hk, C, D)
    return r(B, T, Hq, D), (r(P, Hk, D) if P else None), (r(P, Hk, D) if P else None), r(B, C, Hk, D), r(B, C, Hk, D)


def check(q, pk, pv, k, v, lengths, layout, mask=None, scale=None, causal=True, start=None):
    """One call with weights and one without, both against the reference."""
    if layout == "bhsd":
        cq, cpk, cpv, ck, cv = q, pk, pv, k, v
    else:
        cq, ck, cv = (x.transpose(1, 2) for x in (q, k, v))
        cpk, cpv = (None if x is None else x.transpose(0, 1) for x in (pk, pv))
    ref, ref_w, size, biggest = shared_prefix_ref(cq, cpk, cpv, ck, cv, lengths, mask=mask, scale=scale, causal=causal)
    D, u = q.shape[-1], U[q.dtype]
    e = (D + 8) * 2.0 ** -24 * biggest
    B, Hk, C = ref_w.shape
    start = torch.zeros(B, Hk, C, device=DEV) if start is None else start
    w = start.clone()
    kw = dict(mask=mask, scale=scale, is_causal=causal, layout=layout)
    out = api.shared_prefix_attention(q, pk, pv, k, v, lengths, weights=w, **kw)
    plain = api.shared_prefix_attention(q, pk, pv, k, v, lengths, **kw)
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))
    got = (out if layout == "bhsd" else out.transpose(1, 2)).double()
    bound = u * ref.abs() + (u + 2 * e + 2.0 ** -20) * size + 2.0 ** -24
    assert bool(((got - ref).abs() <= bound).all()), float(((got - ref).abs() - bound).max())
    wb = (2 * e + 2.0 ** -19) * ref_w + 2.0 ** -23 * (start.double() + ref_w)
    off = (w.double() - start.double() - ref_w).abs()
    assert bool((off <= wb).all()), float((off - wb).max())
    assert _lib.device_status(DEV) == 0
    return out


CASES = [
    # (B, T, Hq, Hk, D, P, C, dtype, layout)
    (1, 1, 1, 1, 64, 0, 1, torch.bfloat16, "bhsd"),
    (1, 1, 8, 2, 64, 1, 40, torch.bfloat16, "bhsd"),
    (3, 1, 8, 2, 128, 17, 100, torch.bfloat16, "bshd"),
    (2, 1, 6, 2, 96, 129, 33, torch.float16, "bshd"),
    (2, 1, 4, 1, 256, 300, 50, torch.bfloat16, "bhsd"),
    (5, 3, 4, 2, 128, 64, 70, torch.float16, "bhsd"),
    (2, 7, 14, 2, 64, 130, 48, torch.bfloat16, "bshd"),  # 49 rows a KV head
    (1, 40, 2, 1, 128, 20, 60, torch.bfloat16, "bhsd"),  # a short prompt
    (33, 1, 4, 4, 64, 16, 20, torch.float16, "bhsd"),
    (40, 1, 16, 1, 64, 500, 9, torch.bfloat16, "bshd"),  # 640 rows of the prefix's one head
    (9, 1, 32, 2, 128, 700, 30, torch.bfloat16, "bshd"),
    (20, 1, 20, 2, 256, 257, 12, torch.float16, "bhsd"),
    (24, 2, 12, 2, 96, 400, 10, torch.bfloat16, "bshd"),
    (70, 1, 4, 2, 128, 1025, 5, torch.float16, "bhsd"),
    # Prefixes long enough for the tensor-core kernel: at most 128 rows of a KV head and more,
    # tiles that the prefix's end cuts.
    (12, 1, 16, 2, 64, 6001, 20, torch.bfloat16, "bshd"),
    (300, 1, 2, 2, 64, 2047, 7, torch.float16, "bhsd"),
    (15, 1, 8, 2, 128, 4200, 33, torch.float16, "bshd"),
    (40, 1, 8, 1, 128, 1793, 40, torch.bfloat16, "bhsd"),
    (43, 3, 3, 1, 128, 1409, 9, torch.bfloat16, "bshd"),  # 387 rows: the last slot has none
    (16, 2, 4, 2, 256, 2177, 30, torch.bfloat16, "bshd"),
    (9, 1, 5, 1, 256, 6100, 8, torch.float16, "bhsd"),
    (18, 1, 8, 2, 96, 4608, 11, torch.bfloat16, "bhsd"),
    (100, 2, 1, 1, 96, 3601, 6, torch.float16, "bshd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C,dtype,layout", CASES)
def test_matches_the_formula(B, T, Hq, Hk, D, P, C, dtype, layout):
    g = torch.Generator().manual_seed(B * 100 + P)
    args = make(g, B, T, Hq, Hk, D, P, C, dtype, layout)
    lengths = torch.randint(0, C + 1, (B,), generator=g, dtype=torch.int32)
    lengths[0] = C
    lengths = lengths.to(DEV)
    check(*args, lengths, layout, start=torch.rand(B, Hk, C, generator=g).to(DEV))
    check(*args, lengths, layout, causal=False, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [0, 5, 200])
def test_lengths_of_zero_and_one_and_beyond(P):
    g = torch.Generator().manual_seed(P)
    args = make(g, 6, 2, 4, 2, 64, P, 35, torch.bfloat16, "bshd")
    lengths = torch.tensor([0, 1, 2, 35, -7, 1000], dtype=torch.int32, device=DEV)
    out = check(*args, lengths, "bshd")
    if P == 0:  # no key at all, and the first token of a cache of one
        assert not out[0].any() and not out[1, 0].any() and out[1, 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("Bm,Hm", [(1, 1), (3, 1), (1, 4), (3, 4)])
@pytest.mark.parametrize("P", [0, 40])
def test_masks_rows_left_empty_and_garbage_in_masked_places(Bm, Hm, P):
    """NaN and infinities in K and V wherever no row may look: past the length, after the last
    token, under a mask column of False."""
    g = torch.Generator().manual_seed(11)
    q, pk, pv, k, v = make(g, 3, 3, 4, 2, 128, P, 60, torch.bfloat16, "bhsd")
    mask = torch.rand(Bm, Hm, 3, 60, generator=g) < 0.6
    mask[..., 5] = False
    mask[..., 17] = False
    mask[:, :, 1] = False  # a row that the mask leaves nothing
    mask = mask.to(DEV)
    lengths = torch.tensor([60, 31, 16], dtype=torch.int32, device=DEV)
    for x in (k, v):
        x[:, :, 5], x[:, :, 17] = float("nan"), float("inf")
        x[1, :, 31:], x[2, :, 16:] = float("nan"), -float("inf")
    out = check(q, pk, pv, k, v, lengths, "bhsd", mask=mask)
    check(q, pk, pv, k, v, lengths, "bhsd", mask=mask, causal=False)
    assert bool(torch.isfinite(out).all())
    if P == 0:
        assert not out[:, :, 1].any()
    # A mask given as a view with strides of its own.
    turned = mask.transpose(2, 3).contiguous().transpose(2, 3)
    again = api.shared_prefix_attention(q, pk, pv, k, v, lengths, mask=turned)
    assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
@pytest.mark.parametrize("B,P", [(2, 70), (64, 300), (64, 4500)])
def test_scales(scale, B, P):
    g = torch.Generator().manual_seed(4)
    args = make(g, B, 1, 4, 1, 64, P, 20, torch.float16, "bshd")
    check(*args, torch.full((B,), 20, dtype=torch.int32, device=DEV), "bshd", scale=scale)


@pytest.mark.gpu
def test_growing_logits():
    """Keys in order of rising logits, by a factor that moves the maximum at every tile."""
    g = torch.Generator().manual_seed(6)
    for B, P in ((2, 900), (48, 900), (48, 6000)):
        q, pk, pv, k, v = make(g, B, 1, 4, 1, 64, P, 40, torch.bfloat16, "bhsd")
        q = torch.ones_like(q)
        pk = (torch.arange(P, device=DEV)[None, :, None] * (4.5 / P)).expand_as(pk).to(torch.bfloat16)
        k = k * 0.1 + 4
        check(q, pk, pv, k, v, torch.full((B,), 40, dtype=torch.int32, device=DEV), "bhsd")


@pytest.mark.gpu
@pytest.mark.parametrize("P", [150, 33000])
def test_strided_and_unaligned_inputs_give_the_same_bits(P):
    g = torch.Generator().manual_seed(8)
    q, pk, pv, k, v = make(g, 3, 2, 4, 2, 64, P, 50, torch.bfloat16, "bhsd")
    lengths = torch.tensor([50, 20, 2], dtype=torch.int32, device=DEV)
    want = api.shared_prefix_attention(q, pk, pv, k, v, lengths)

    def shifted(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape)
        return y.copy_(x)

    def padded(x):
        y = torch.full((*x.shape[:-1], 80), float("nan"), dtype=x.dtype, device=DEV)[..., 8:72]
        return y.copy_(x)

    def seq_first(x):
        return x.transpose(-3, -2).contiguous().transpose(-3, -2)

    for f in (shifted, padded, seq_first):
        assert torch.equal(api.shared_prefix_attention(f(q), pk, pv, k, v, lengths), want)
        assert torch.equal(api.shared_prefix_attention(q, f(pk), f(pv), f(k), f(v), lengths), want)
    # One head of the prefix and of the caches for all (a stride of 0).
    one = [x[..., :1, :, :].expand(x.shape) for x in (pk, pv, k, v)]
    whole = [x.contiguous() for x in one]
    assert torch.equal(api.shared_prefix_attention(q, *one, lengths), api.shared_prefix_attention(q, *whole, lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("P", [600, 2000])
def test_repeats_bit_for_bit_in_a_graph_and_on_another_stream(P):
    g = torch.Generator().manual_seed(9)
    q, pk, pv, k, v = make(g, 40, 1, 8, 2, 128, P, 90, torch.bfloat16, "bshd")
    lengths = torch.randint(1, 91, (40,), generator=g, dtype=torch.int32).to(DEV)
    w0 = torch.zeros(40, 2, 90, device=DEV)
    call = lambda w: api.shared_prefix_attention(q, pk, pv, k, v, lengths, weights=w, layout="bshd")  # noqa: E731
    w = w0.clone()
    want = call(w)
    for _ in range(5):
        w1 = w0.clone()
        assert torch.equal(call(w1), want) and torch.equal(w1, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1 = w0.clone()
        other = call(w1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want) and torch.equal(w1, w)
    w1 = w0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(w1)
    w1.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(w1, w)


@pytest.mark.gpu
@pytest.mark.parametrize("B,P", [(2, 0), (40, 500), (40, 2000)])
def test_inputs_changed_in_place_between_calls(B, P):
    """Back-to-back calls with no synchronisation, each after kernels that rewrite lengths, query,
    caches and mask in the same memory: every call sees its own inputs."""
    g = torch.Generator().manual_seed(10)
    q, pk, pv, k, v = make(g, B, 2, 8, 2, 64, P, 70, torch.bfloat16, "bhsd")
    steps = []
    for i in range(6):
        steps.append((torch.randn(q.shape, generator=g).to(q), torch.randn(k.shape, generator=g).to(k),
                      torch.randint(0, 71, (B,), generator=g, dtype=torch.int32).to(DEV),
                      (torch.rand(B, 1, 2, 70, generator=g) < 0.7).to(DEV)))
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    mask = torch.zeros(B, 1, 2, 70, dtype=torch.bool, device=DEV)
    w = torch.zeros(B, 2, 70, device=DEV)
    got = []
    for q1, k1, n1, m1 in steps:
        for dst, src in ((q, q1), (k, k1), (lengths, n1), (mask, m1)):
            dst.copy_(src)
        w.zero_()
        got.append((api.shared_prefix_attention(q, pk, pv, k, v, lengths, mask=mask, weights=w), w.clone()))
    for (q1, k1, n1, m1), (out, w1) in zip(steps, got):
        torch.cuda.synchronize()
        w.zero_()
        again = api.shared_prefix_attention(q1, pk, pv, k1, v, n1, mask=m1, weights=w)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(w1, w)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    store = torch.empty(2 ** 31 + 65536, dtype=torch.bfloat16, device=DEV)
    k = store.as_strided((2, 1, 200, 64), (2 ** 31 + 8, 64 * 200, 64, 1))
    g = torch.Generator().manual_seed(0)
    q, pk, pv, k0, _ = make(g, 2, 1, 2, 1, 64, 30, 200, torch.bfloat16, "bhsd")
    k.copy_(k0)
    lengths = torch.tensor([200, 150], dtype=torch.int32, device=DEV)
    want = api.shared_prefix_attention(q, pk, pv, k0, k0, lengths)
    assert torch.equal(api.shared_prefix_attention(q, pk, pv, k, k, lengths), want)
