"""Attention over own caches in 8 bits (and a shared prefix in 16) against the 64-bit formula of the
values that the caches hold.

Weights are rounded to fp16 before the product with V (2^-11 p |v| for each key, and 2^-25 of the
largest |v| for each of K keys whose weight falls below fp16's normal range), those of a prefix to the
type of the query (u), the result once (u |o|); queries and codes go to the products exactly (what
falls below fp16's steps there is under 2^-39 of the row's largest); the logits carry the error of a
32-bit dot product of D terms, e = (D + 16) 2^-24 max sum|q k| |scale| plus the exponential's 2^-21,
twice: |o - o64| <= u |o64| + (up + 2 e + 2^-20) sum p |v| + 2^-25 K max|v| + 2^-24, up = 2^-11, with a
prefix u."""

from __future__ import annotations

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import BLOCK, values_ref
from oracle.serving import shared_prefix_ref

DEV = torch.device("cuda", 0)
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def codes(g, shape, code):
    if code == INT8:
        return torch.randint(-127, 128, shape, generator=g).to(torch.int8).to(DEV)
    return (torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(E4M3).to(DEV)


def make(g, B, T, Hq, Hk, D, P, C, dtype, code, layout):
    r = lambda *s: torch.randn(s, generator=g).to(dtype).to(DEV)  # noqa: E731
    seq = lambda n, H: (B, H, n, D) if layout == "bhsd" else (B, n, H, D)  # noqa: E731
    pre = (lambda: r(Hk, P, D) if layout == "bhsd" else r(P, Hk, D)) if P else lambda: None
    # Not powers of two only: any scales can be read.
    scale = lambda: (torch.exp2(torch.rand(B, Hk, -(-C // BLOCK), generator=g) * 3 - 8)).to(DEV)  # noqa: E731
    return dict(q=r(*seq(T, Hq)), pk=pre(), pv=pre(), k=codes(g, seq(C, Hk), code), v=codes(g, seq(C, Hk), code), ks=scale(), vs=scale())


def call(a, lengths, layout, **kw):
    return api.shared_prefix_attention(a["q"], a["pk"], a["pv"], a["k"], a["v"], lengths, key_scale=a["ks"], value_scale=a["vs"],
                                       layout=layout, **kw)


def check(a, lengths, layout, mask=None, scale=None, causal=True):
    c = {n: x if x is None or layout == "bhsd" or n in ("ks", "vs") else x.transpose(0, 1) if x.dim() == 3 else x.transpose(1, 2)
         for n, x in a.items()}
    C = c["k"].shape[2]
    k, v = (values_ref(c[n], c[n + "s"], lengths.clamp(0, C)) for n in ("k", "v"))
    ref, _, size, biggest = shared_prefix_ref(c["q"], c["pk"], c["pv"], k, v, lengths, mask=mask, scale=scale, causal=causal)
    D, u = c["q"].shape[3], U[c["q"].dtype]
    e = (D + 16) * 2.0 ** -24 * biggest
    up = 2.0 ** -11 if c["pk"] is None else u
    out = call(a, lengths, layout, mask=mask, scale=scale, is_causal=causal)
    got = (out if layout == "bhsd" else out.transpose(1, 2)).double()
    largest = float(v.abs().nan_to_num(0.0, 0.0, 0.0).max())
    bound = u * ref.abs() + (up + 2 * e + 2.0 ** -20) * size + 2.0 ** -25 * C * largest + 2.0 ** -24
    off = (got - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())
    assert _lib.device_status(DEV) == 0
    return out


CASES = [
    # (B, T, Hq, Hk, D, P, C, dtype, code, layout)
    (1, 1, 1, 1, 64, 0, 1, BF16, E4M3, "bhsd"),
    (1, 1, 8, 2, 64, 0, 140, BF16, INT8, "bhsd"),
    (3, 1, 8, 2, 128, 0, 100, BF16, E4M3, "bshd"),
    (2, 1, 6, 2, 96, 0, 133, FP16, E4M3, "bshd"),
    (2, 1, 6, 2, 96, 40, 70, BF16, INT8, "bhsd"),
    (2, 1, 4, 1, 256, 0, 90, BF16, E4M3, "bhsd"),
    (5, 3, 4, 2, 128, 0, 70, FP16, INT8, "bhsd"),
    (2, 7, 14, 2, 64, 0, 148, BF16, E4M3, "bshd"),  # 49 rows a KV head
    (1, 40, 2, 1, 128, 0, 60, BF16, INT8, "bhsd"),  # a short prompt
    (2, 5, 8, 2, 256, 0, 77, FP16, INT8, "bshd"),  # 20 rows
    (2, 9, 4, 2, 256, 0, 65, BF16, E4M3, "bhsd"),
    (33, 1, 4, 4, 64, 0, 20, FP16, E4M3, "bhsd"),
    (9, 1, 32, 2, 128, 300, 130, BF16, E4M3, "bshd"),
    (20, 1, 20, 2, 256, 257, 72, FP16, INT8, "bhsd"),
    (12, 1, 16, 2, 64, 2001, 90, BF16, INT8, "bshd"),
    (3, 2, 12, 2, 96, 400, 66, BF16, E4M3, "bshd"),
    (2, 1, 16, 1, 128, 0, 3000, BF16, E4M3, "bhsd"),
    (140, 1, 2, 1, 128, 0, 200, FP16, E4M3, "bshd"),
    (2, 3, 16, 2, 128, 0, 150, BF16, E4M3, "bshd"),  # 24 rows
    (1, 5, 14, 1, 96, 0, 130, FP16, INT8, "bhsd"),  # 70 rows, the last tile with 6
    (2, 1, 33, 1, 64, 0, 200, FP16, E4M3, "bhsd"),  # 33 rows
    (3, 2, 12, 1, 96, 0, 65, BF16, E4M3, "bshd"),
    (2, 9, 8, 4, 64, 70, 100, BF16, INT8, "bshd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C,dtype,code,layout", CASES)
def test_matches_the_formula(B, T, Hq, Hk, D, P, C, dtype, code, layout):
    g = torch.Generator().manual_seed(B * 100 + P + C)
    a = make(g, B, T, Hq, Hk, D, P, C, dtype, code, layout)
    lengths = torch.randint(0, C + 1, (B,), generator=g, dtype=torch.int32)
    lengths[0] = C
    lengths = lengths.to(DEV)
    check(a, lengths, layout)
    check(a, lengths, layout, causal=False, scale=0.03)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_around_blocks_and_beyond(code, D):
    g = torch.Generator().manual_seed(D)
    a = make(g, 12, 2, 4, 2, D, 0, 130, BF16, code, "bshd")
    lengths = torch.tensor([0, 1, 2, 16, 63, 64, 65, 127, 128, 130, -7, 1000], dtype=torch.int32, device=DEV)
    out = check(a, lengths, "bshd")
    assert not out[0].any() and not out[1, 0].any() and out[1, 1].any()  # no key at all, and the first of two tokens


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Bm,Hm,T", [(1, 1, 3), (3, 1, 3), (1, 4, 9), (3, 4, 9)])
def test_masks_rows_left_empty_and_garbage_in_masked_places(Bm, Hm, T, D, code):
    """NaN codes and scales wherever no row may look: past the length, under mask columns of False,
    a whole block of which has a NaN scale."""
    g = torch.Generator().manual_seed(11)
    a = make(g, 3, T, 4, 2, D, 0, 200, BF16, code, "bhsd")
    mask = torch.rand(Bm, Hm, T, 200, generator=g) < 0.6
    mask[..., 5] = False
    mask[..., 64:128] = False
    mask[:, :, 1] = False  # a row that the mask leaves nothing
    mask = mask.to(DEV)
    lengths = torch.tensor([200, 31, 66], dtype=torch.int32, device=DEV)
    for n in ("k", "v"):
        c = a[n].view(torch.uint8)
        c[:, :, 5], c[1, :, 31:], c[2, :, 66:] = 0x7f, 0xff, 0x7f
        a[n + "s"][:, :, 1] = float("nan")
        a[n + "s"][1, :, 1:] = float("inf")
    if code == E4M3:
        ref = dict(a, **{n: a[n].to(torch.float32).nan_to_num(0.0).to(E4M3) for n in ("k", "v")})
    else:
        ref = dict(a)
    ref.update({n: a[n].nan_to_num(1.0, posinf=1.0) for n in ("ks", "vs")})
    for causal in (True, False):
        want = check(ref, lengths, "bhsd", mask=mask, causal=causal)
        got = call(a, lengths, "bhsd", mask=mask, is_causal=causal)
        assert torch.equal(got, want) and bool(torch.isfinite(got).all()) and not got[:, :, 1].any()
    turned = mask.transpose(2, 3).contiguous().transpose(2, 3)  # strides of its own
    assert torch.equal(call(a, lengths, "bhsd", mask=turned, is_causal=False), got)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_what_a_row_sees_of_nan_is_nan_and_nothing_else(code):
    """A NaN scale of keys or of values reaches the rows that see the block, a query that is not
    finite its own rows."""
    g = torch.Generator().manual_seed(12)
    a = make(g, 4, 2, 4, 2, 128, 0, 200, BF16, code, "bhsd")
    lengths = torch.tensor([200, 200, 64, 65], dtype=torch.int32, device=DEV)  # the last: token 0 ends before the block
    a["ks"][0, 0, 2] = float("nan")
    a["vs"][:, :, 1] = float("nan")
    a["vs"][0, :, 1] = 1.0
    a["q"][1, 3, 1, 7] = float("inf")
    a["vs"][1, :, 1] = 1.0
    out = call(a, lengths, "bhsd")
    bad = torch.isnan(out).all(-1)
    assert torch.equal(bad, torch.isnan(out).any(-1))
    assert bad[0].tolist() == [[True, True], [True, True], [False, False], [False, False]]
    assert bad[1].tolist() == [[False, False], [False, False], [False, False], [False, True]]
    assert not bad[2].any() and bad[3].tolist() == [[False, True]] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_a_block_of_large_scale_without_weight_costs_no_bits(code):
    """Values a million times larger under keys of logit 0, where the other blocks' keys lie along the
    query and get all the weight; and a block whose values have scale 0.  Weights below 2^-43 that are
    rounded to 0 lose at most 64 * 2^-43 * 2^20 = 2^-17 of the others' largest |v|: no more than the
    bound allows for K = 256 keys of that size."""
    g = torch.Generator().manual_seed(13)
    a = make(g, 2, 1, 4, 1, 64, 0, 256, FP16, code, "bhsd")
    a["vs"][:, :, 1] *= 2.0 ** 20
    a["vs"][:, :, 2] = 0.0
    a["q"], a["ks"][:] = a["q"][:, :1].repeat(1, 4, 1, 1) * 0.3, 1.0
    along = a["q"][:, 0, 0].float() * 60
    k = along.round().clamp(-127, 127).to(INT8) if code == INT8 else along.to(E4M3)
    a["k"] = k[:, None, None].view(torch.uint8).repeat(1, 1, 256, 1)
    a["k"][:, :, 64:128] = 0
    a["k"] = a["k"].view(code)
    lengths = torch.tensor([256, 192], dtype=torch.int32, device=DEV)
    k, v = (values_ref(a[n], a[n + "s"], lengths) for n in ("k", "v"))
    assert float((k[:, 0, 0] * a["q"][:, 0, 0].double()).sum(-1).min()) * 64 ** -0.5 > 30  # e^-30 < 2^-43
    ref, _, size, biggest = shared_prefix_ref(a["q"], None, None, k, v, lengths)
    e = (64 + 16) * 2.0 ** -24 * biggest
    bound = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2 * e + 2.0 ** -20) * size + 2.0 ** -25 * 256 * float(v[:, :, :64].abs().max()) + 2.0 ** -24
    off = (call(a, lengths, "bhsd").double() - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_queries_of_any_size(dtype):
    """Rows whose largest element is far from 1 go to the products by a power of two of their own."""
    g = torch.Generator().manual_seed(14)
    a = make(g, 2, 4, 2, 1, 64, 0, 100, dtype, E4M3, "bhsd")
    for t, f in enumerate([2.0 ** -13, 2.0 ** 8, 0.0, 2.0 ** -5]):
        a["q"][:, :, t] *= f
    a["q"][0, 0, 1, 3], a["q"][0, 0, 3, :] = 60000.0, 0.0
    a["ks"] *= 2.0 ** -9
    lengths = torch.tensor([100, 50], dtype=torch.int32, device=DEV)
    check(a, lengths, "bhsd", scale=0.01)
    if dtype == BF16:
        b = dict(a, q=a["q"] * 2.0 ** 100, ks=a["ks"] * 2.0 ** -100)
        check(b, lengths, "bhsd", scale=0.01)
        b = dict(a, q=a["q"] * 2.0 ** -100, ks=a["ks"] * 2.0 ** 100)
        check(b, lengths, "bhsd", scale=0.01)


@pytest.mark.gpu
def test_strided_unaligned_other_stream_graph_and_repeats():
    g = torch.Generator().manual_seed(15)
    a = make(g, 3, 1, 8, 2, 128, 0, 150, BF16, E4M3, "bshd")
    lengths = torch.tensor([150, 1, 77], dtype=torch.int32, device=DEV)
    want = call(a, lengths, "bshd")
    assert torch.equal(call(a, lengths, "bshd"), want)
    b = {n: None if x is None else x.transpose(1, 2) if n in "qkv" else x for n, x in a.items()}
    assert torch.equal(call(b, lengths, "bhsd").transpose(1, 2), want)
    off = torch.zeros(3, 150, 2, 129, dtype=torch.uint8, device=DEV)[..., 1:]
    off.copy_(a["k"].view(torch.uint8))
    wide = torch.zeros(3, 2, 7, device=DEV)
    wide[..., 2:5].copy_(a["vs"])
    odd = torch.zeros(a["q"].numel() + 1, dtype=BF16, device=DEV)[1:].view(a["q"].shape)
    odd.copy_(a["q"])
    assert torch.equal(call(dict(a, k=off.view(E4M3), vs=wide[..., 2:5], q=odd), lengths, "bshd"), want)
    one = call(dict(a, k=a["k"][:1].expand(3, -1, -1, -1), ks=a["ks"][:1].expand(3, -1, -1)), lengths, "bshd")  # keys shared
    each = call(dict(a, k=a["k"].view(torch.uint8)[:1].repeat(3, 1, 1, 1).view(E4M3), ks=a["ks"][:1].repeat(3, 1, 1)), lengths, "bshd")
    assert torch.equal(one, each)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(dict(a, q=a["q"] * 1), lengths, "bshd") for _ in range(3)]
        here = call(a, lengths, "bshd")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in (*got, here))
    graphs, outs, q, n = [], [], a["q"].clone(), lengths.clone()
    for _ in range(2):  # two graphs of the same call, replayed in turn and together
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(dict(a, q=q), n, "bshd"))
        graphs.append(graph)
    n.copy_(torch.tensor([3, 150, 64], dtype=torch.int32))
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    again = call(a, n, "bshd")
    assert torch.equal(outs[0], again) and torch.equal(outs[1], again)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The second request's codes lie past 2^32 bytes, and slots of one request past 2^31."""
    g = torch.Generator().manual_seed(16)
    a = make(g, 2, 1, 4, 1, 64, 0, 70, BF16, INT8, "bhsd")
    lengths = torch.tensor([70, 66], dtype=torch.int32, device=DEV)
    want = call(a, lengths, "bhsd")
    store = torch.zeros(2 ** 32 + 2 * 70 * 64 + 64, dtype=torch.int8, device=DEV)
    big = store.as_strided((2, 1, 70, 64), (2 ** 32 + 64, 70 * 64, 64, 1))
    big.copy_(a["k"])
    assert torch.equal(call(dict(a, k=big), lengths, "bhsd"), want)
    far = store.as_strided((2, 1, 70, 64), (64, 128, 2 ** 25 + 128, 1))
    far.copy_(a["v"])
    assert torch.equal(call(dict(a, v=far), lengths, "bhsd"), want)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_a_run_of_decode_steps(code):
    """Norm, turn and append into 8-bit caches, attention over a prefix and them, step after step, as a
    model would; every step against the 64-bit formula of what the caches hold, which in turn is
    within a code of what was appended; at last a request's cache becomes the next prefix."""
    g = torch.Generator().manual_seed(17)
    B, Hq, Hk, D, P, C = 3, 8, 2, 128, 50, 100
    rope = api.MultiAxisRotary(D, (16, 24, 24))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(DEV) for _ in range(2)]
    r = lambda *s: torch.randn(s, generator=g).to(BF16).to(DEV)  # noqa: E731
    pk, pv = rope(r(1, P, Hq, D), r(1, P, Hk, D), torch.arange(P, device=DEV).expand(3, 1, P), query_norm=w[0], key_norm=w[1],
                  layout="bshd")[1][0], r(P, Hk, D)
    kc, vc = (torch.empty(B, C, Hk, D, dtype=code, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(B, Hk, 2, device=DEV) for _ in range(2))
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for step, T in enumerate([58, 1, 1, 9, 1, 20]):
        q, k, v = r(B, T, Hq, D), r(B, T, Hk, D), r(B, T, Hk, D)
        pos = (P + lengths.long()[None, :, None] + torch.arange(T, device=DEV)).expand(3, B, T)
        q, lengths = rope.append(q, k, v, pos, kc, vc, lengths, query_norm=w[0], key_norm=w[1], key_scale=ks, value_scale=vs,
                                 layout="bshd")
        held = api.cache_values(vc, vs, lengths, layout="bshd")
        n = int(lengths[0])
        assert float((held[:, n - T:n].double() - v.double()).abs().max()) <= float(v.abs().max()) * 2.0 ** -4
        if T < 10:
            check(dict(q=q, pk=pk, pv=pv, k=kc, v=vc, ks=ks, vs=vs), lengths, "bshd")
    n = int(lengths[1])
    pk, pv = (api.cache_values(c, s, lengths, layout="bshd")[1, :n] for c, s in ((kc, ks), (vc, vs)))
    check(dict(q=q[:, :1].contiguous(), pk=pk, pv=pv, k=kc, v=vc, ks=ks, vs=vs), lengths * 0 + 3, "bshd")
    assert _lib.device_status(DEV) == 0
