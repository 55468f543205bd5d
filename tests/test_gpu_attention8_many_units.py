"""Attention over caches in 8 bits where every warp takes many units: rings that go round, maxima that
rise and fall from unit to unit, weights and scales far apart.

The bound is that of ``test_gpu_attention8`` (fp16 weights 2^-11 of p |v|, with a prefix the query's u;
logits off by e = (D + 16) 2^-24 max sum|q k| |scale| and the exponential's 2^-21, twice; the result once,
u), but for small weights: the largest weight that a warp gives the product with V is 1 or more, so fp16's
least half step, 2^-25, is at most that of the largest p z (z a block's scale of V), for each of K keys,
times the largest code."""

from __future__ import annotations

import math

import pytest
import torch

from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import BLOCK, LARGEST, values_ref
from test_gpu_attention8 import BF16, DEV, E4M3, FP16, INT8, U, call


def codes(g, shape, code):
    if code == INT8:
        return torch.randint(-127, 128, shape, generator=g, device=DEV).to(torch.int8)
    return (torch.randn(shape, generator=g, device=DEV) * 100).clamp(-448, 448).to(E4M3)


def make(seed, B, T, Hq, Hk, D, P, C, dtype, code, layout):
    """As in ``test_gpu_attention8``, made on the GPU."""
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    seq = lambda n, H: (B, H, n, D) if layout == "bhsd" else (B, n, H, D)  # noqa: E731
    pre = (lambda: r(Hk, P, D) if layout == "bhsd" else r(P, Hk, D)) if P else lambda: None
    scale = lambda: torch.exp2(torch.rand(B, Hk, -(-C // BLOCK), generator=g, device=DEV) * 3 - 8)  # noqa: E731
    return dict(q=r(*seq(T, Hq)), pk=pre(), pv=pre(), k=codes(g, seq(C, Hk), code), v=codes(g, seq(C, Hk), code), ks=scale(), vs=scale())


def formula(a, lengths, layout, mask=None, scale=None, causal=True):
    """(out, sum of p |v|, largest p z, largest sum of |q k| * |scale|) in 64 bits, canonical layout."""
    swap = lambda x: x if layout == "bhsd" else x.transpose(1, 2)  # noqa: E731
    q, kc, vc = swap(a["q"]).double(), swap(a["k"]), swap(a["v"])
    B, Hq, T, D = q.shape
    Hk, C = kc.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    pk, pv = (None if a[n] is None else (a[n] if layout == "bhsd" else a[n].transpose(0, 1)).double() for n in ("pk", "pv"))
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    size, top, biggest = torch.zeros_like(out), torch.zeros(B, Hq, T, 1, dtype=torch.float64, device=DEV), 0.0
    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), C)
        one = torch.tensor([n])
        k, v = (values_ref(x[b:b + 1], s[b:b + 1], one.to(DEV))[0, :, :n] for x, s in ((kc, a["ks"]), (vc, a["vs"])))
        z = a["vs"][b].double().repeat_interleave(BLOCK, 1)[:, :n]
        rows = q[b].reshape(Hk, Hq // Hk, T, D)  # [Hk, G, T, D]
        seen = torch.ones(T, n, dtype=torch.bool, device=DEV)
        if causal:
            seen = torch.arange(n, device=DEV)[None] < n - T + 1 + torch.arange(T, device=DEV)[:, None]
        seen = seen.expand(Hk, Hq // Hk, T, n)
        if mask is not None:
            seen = seen & mask[b % mask.shape[0], :, :, :n].expand(Hq, T, n).reshape(Hk, Hq // Hk, T, n)
        some = seen.any(2).any(1)  # [Hk, n]: others may hold anything
        k, v = (x.masked_fill(~some[..., None], 0.0) for x in (k, v))
        z = z.masked_fill(~some, 0.0)
        if pk is not None:
            P = pk.shape[1]
            k, v, z = torch.cat([pk, k], 1), torch.cat([pv, v], 1), torch.cat([torch.zeros(Hk, P, device=DEV), z], 1)
            seen = torch.cat([seen.new_ones(*seen.shape[:3], P), seen], 3)
        if not k.shape[1]:
            continue
        x = torch.einsum("hgtd,hnd->hgtn", rows, k) * scale
        biggest = max(biggest, float(torch.einsum("hgtd,hnd->hgtn", rows.abs(), k.abs()).max()) * abs(scale))
        x = x.masked_fill(~seen, -math.inf)
        p = torch.softmax(x, 3).nan_to_num(0.0)  # rows that see nothing
        out[b] = torch.einsum("hgtn,hnd->hgtd", p, v).reshape(Hq, T, D)
        size[b] = torch.einsum("hgtn,hnd->hgtd", p, v.abs()).reshape(Hq, T, D)
        top[b] = (p * z[:, None, None]).amax(3).reshape(Hq, T, 1)
    return out, size, top, biggest


def check(a, lengths, layout, mask=None, scale=None, causal=True):
    ref, size, top, biggest = formula(a, lengths, layout, mask, scale, causal)
    dtype, D, C = a["q"].dtype, a["q"].shape[3], a["k"].shape[2 if layout == "bhsd" else 1]
    e = (D + 16) * 2.0 ** -24 * biggest
    up = 2.0 ** -11 if a["pk"] is None else U[dtype]
    out = call(a, lengths, layout, mask=mask, scale=scale, is_causal=causal)
    got = (out if layout == "bhsd" else out.transpose(1, 2)).double()
    bound = U[dtype] * ref.abs() + (up + 2 * e + 2.0 ** -20) * size + 2.0 ** -25 * C * LARGEST[a["k"].dtype] * top + 2.0 ** -24
    off = (got - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())
    for _ in range(2):  # the same bits every time
        assert torch.equal(call(a, lengths, layout, mask=mask, scale=scale, is_causal=causal), out)
    assert _lib.device_status(DEV) == 0
    return out


def units_of_a_warp(lengths, C, R, D, Hk):
    """Units (of 64 to 16 keys, by the head dim) that a warp takes on average."""
    keys, ctas = {64: 64, 96: 32, 128: 32, 256: 16}[D], 3 if R <= 8 and D <= 128 else 2
    units = sum(-(-min(n, C) // keys) for n in lengths.tolist()) * Hk * -(-R // 16)
    return units / (4 * ctas * torch.cuda.get_device_properties(DEV).multi_processor_count)


CASES = [
    # (B, T, Hq, Hk, D, P, C, dtype, code, layout)
    (64, 1, 32, 8, 128, 0, 2048, BF16, E4M3, "bshd"),
    (64, 1, 32, 8, 128, 0, 2048, FP16, INT8, "bhsd"),
    (64, 2, 16, 8, 64, 0, 4099, BF16, E4M3, "bhsd"),
    (48, 1, 64, 1, 64, 0, 8191, BF16, INT8, "bshd"),  # 64 rows: four row tiles
    (96, 1, 40, 2, 64, 0, 4001, FP16, E4M3, "bshd"),  # 20 rows
    (24, 6, 16, 4, 256, 0, 2050, BF16, INT8, "bshd"),  # 24 rows
    (48, 1, 16, 4, 256, 0, 2050, FP16, E4M3, "bhsd"),
    (128, 3, 16, 4, 96, 0, 1500, BF16, E4M3, "bshd"),  # 12 rows
    (96, 1, 18, 6, 96, 0, 2100, FP16, INT8, "bhsd"),  # 3 rows
    (200, 2, 8, 4, 128, 0, 1300, FP16, E4M3, "bshd"),  # lengths past 128 requests are read from memory
    (64, 1, 32, 8, 128, 700, 2048, BF16, E4M3, "bshd"),
    (96, 2, 32, 4, 64, 2000, 4000, FP16, INT8, "bhsd"),  # 16 rows
    (24, 3, 24, 4, 256, 300, 1500, BF16, E4M3, "bshd"),  # 18 rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C,dtype,code,layout", CASES)
def test_rings_go_round(B, T, Hq, Hk, D, P, C, dtype, code, layout):
    g = torch.Generator().manual_seed(B * 100 + P + C)
    a = make(B * 100 + P + C, B, T, Hq, Hk, D, P, C, dtype, code, layout)
    lengths = torch.randint(0, C + 1, (B,), generator=g, dtype=torch.int32)
    lengths[0], lengths[1] = C, 0
    assert units_of_a_warp(lengths, C, T * Hq // Hk, D, Hk) >= 6  # rings of 2 or 3
    check(a, lengths.to(DEV), layout)
    check(a, lengths.to(DEV), layout, causal=False, scale=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("B,T,Hq,Hk,D,P,C", [(64, 2, 16, 8, 64, 0, 4000), (64, 3, 16, 4, 128, 0, 3000), (96, 3, 8, 4, 96, 90, 3000),
                                             (64, 2, 16, 4, 256, 0, 1500)])
def test_masks_that_leave_whole_units_empty(B, T, Hq, Hk, D, P, C, code):
    """Stretches that no row sees, with NaN codes and scales there and past the lengths: V is cleared in a
    stage that is filled again behind it."""
    g = torch.Generator().manual_seed(C + D)
    a = make(C + D, B, T, Hq, Hk, D, P, C, BF16, code, "bhsd")
    blocks = -(-C // BLOCK)
    dark = torch.rand(B, 1, 1, blocks, generator=g) < 0.4
    mask = (torch.rand(B, 1, T, C, generator=g) < 0.7) & ~dark.repeat_interleave(BLOCK, 3)[..., :C]
    mask[2] = False  # a request whose mask leaves nothing
    lengths = torch.randint(1, C + 1, (B,), generator=g, dtype=torch.int32)
    assert units_of_a_warp(lengths, C, T * Hq // Hk, D, Hk) >= 6
    nowhere = ~mask.any(2).view(B, 1, C, 1) | (torch.arange(C) >= lengths[:, None]).view(B, 1, C, 1)
    for n in ("k", "v"):
        a[n].view(torch.uint8).masked_fill_(nowhere.to(DEV), 0x7f)
        a[n + "s"].masked_fill_(dark[:, 0, 0, None].expand_as(a[n + "s"]).to(DEV), float("nan"))
    for causal in (True, False):
        out = check(a, lengths.to(DEV), "bhsd", mask=mask.to(DEV), causal=causal)
        assert P or not out[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("D,Hq,Hk", [(64, 16, 2), (128, 8, 2), (128, 20, 2), (256, 24, 2)])
@pytest.mark.parametrize("swing", [3.0, 30.0])
def test_logits_and_scales_that_rise_and_fall(swing, D, Hq, Hk, code):
    """Logits of up to +-swing (in powers of two) and scales of V of 2^+-swing, both slowly along the keys:
    maxima that follow at once, and ones that lag within their slack."""
    g = torch.Generator().manual_seed(int(swing) + D)
    B, C = 112, 6000 * 64 // D
    a = make(D, B, 1, Hq, Hk, D, 0, C, BF16, code, "bhsd")
    sign = (torch.randint(0, 2, (D,), generator=g) * 2 - 1).float()
    part = torch.linspace(-1, 1, Hq).to(BF16).float()  # heads whose logits rise, and fall, and do neither
    a["q"] = (sign * part[:, None]).to(BF16).to(DEV)[None, :, None].repeat(B, 1, 1, 1)
    j = torch.arange(C)
    at = (96 * torch.sin(j / 333 + torch.arange(B)[:, None])).round()[:, None, :, None] * sign  # [B, 1, C, D]
    at = at.to(DEV).expand(B, Hk, C, D)
    a["k"] = at.to(torch.int8).contiguous() if code == INT8 else at.to(E4M3)
    a["ks"].fill_(1.0)
    z = swing * torch.sin(torch.arange(a["vs"].shape[2]) / 7.0 + torch.arange(B)[:, None]) - 4
    a["vs"] = torch.exp2(z)[:, None].expand(B, Hk, -1).contiguous().to(DEV)
    lengths = torch.randint(C // 2, C + 1, (B,), generator=g, dtype=torch.int32)
    assert units_of_a_warp(lengths, C, Hq // Hk, D, Hk) >= 6
    check(a, lengths.to(DEV), "bhsd", scale=swing * math.log(2) / (96 * D))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("D,Hq", [(64, 1), (64, 8), (64, 16), (96, 8), (128, 8), (128, 16), (256, 8), (256, 16)])
@pytest.mark.parametrize("below,above", [(120.5, 28), (125.5, 33)])
def test_scales_of_values_far_apart(below, above, D, Hq, code):
    """A block of values of 2^-100 whose logits are 0, then one of 2^above whose logits are -below (in powers
    of two): the second has 2^7.5 times the first one's part of the output, although its probabilities are
    near 32 bits' least.  Every request holds the same, and the line is divided between and within them:
    the bound holds wherever.  (Row tiles that are full: the rows beside have logits of 0.)"""
    B, C = 2400, 128
    g = torch.Generator(DEV).manual_seed(5)
    v = codes(g, (1, 1, C, D), code)
    k = torch.zeros(1, 1, C, D, device=DEV)
    k[:, :, 64:, 0] = -96.0
    k = k.to(torch.int8) if code == INT8 else k.to(E4M3)
    q = torch.zeros(1, Hq, 1, D, dtype=BF16, device=DEV)
    q[..., 0] = 1.0
    ks, vs = torch.tensor([1.0, below / 96], device=DEV), torch.tensor([2.0 ** -100, 2.0 ** above], device=DEV)
    every = lambda x: x.view(torch.uint8).repeat(B, 1, 1, 1).view(x.dtype)  # noqa: E731
    a = dict(q=q.repeat(B, 1, 1, 1), pk=None, pv=None, k=every(k), v=every(v), ks=ks.repeat(B, 1, 1), vs=vs.repeat(B, 1, 1))
    lengths = torch.full((B,), C, dtype=torch.int32, device=DEV)
    out = call(a, lengths, "bhsd", scale=math.log(2)).double()
    one = {n: None if x is None else x[:1] for n, x in a.items()}
    ref, size, top, biggest = formula(one, lengths[:1], "bhsd", scale=math.log(2))
    e = (D + 16) * 2.0 ** -24 * biggest
    bound = U[BF16] * ref.abs() + (2.0 ** -11 + 2 * e + 2.0 ** -20) * size + 2.0 ** -25 * C * LARGEST[code] * top
    off = ((out - ref).abs() / bound).amax((1, 2, 3))
    assert bool((off <= 1).all()), (float(off.max()), int(off.argmax()))


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_logits_and_scales_that_are_no_powers_of_two(dtype, code):
    """Equal keys: every logit is the same, 1.2 million, so the output is the values' mean, whatever a logit's
    error.  The exponents that weights are made of are differences of logits, and keep their bits."""
    a = make(6, 3, 1, 4, 2, 64, 0, 1000, dtype, code, "bhsd")
    a["q"].fill_(64.0)
    a["k"] = torch.full(a["k"].shape, 96.0, device=DEV).to(code)
    a["v"] = (a["v"].view(torch.uint8) & 0x7F).view(code)  # positive
    a["ks"].fill_(2.0)
    lengths = torch.tensor([1000, 300, 65], dtype=torch.int32)
    out = call(a, lengths.to(DEV), "bhsd", scale=1.0).double()
    for b, n in enumerate(lengths.tolist()):
        v = values_ref(a["v"][b:b + 1], a["vs"][b:b + 1], lengths[b:b + 1].to(DEV))[0, :, :n].repeat_interleave(2, 0)
        mean, size = v.mean(1, keepdim=True), v.abs().mean(1, keepdim=True)
        bound = U[dtype] * mean.abs() + (2.0 ** -11 + 2.0 ** -20) * size + 2.0 ** -25 * 448 * float(a["vs"].max()) + 2.0 ** -24
        off = (out[b] - mean).abs() - bound
        assert bool((off <= 0).all()), (b, float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 12), (256, 4)])
@pytest.mark.parametrize("power", [-126, -118, 100])
def test_values_of_any_size(power, D, Hq):
    """Scales of V down to the least that appending writes; steps of bf16's least exponent, and of partial
    rows in 32 bits, beside the bound."""
    a = make(7, 12, 1, Hq, 1, D, 0, 1000, BF16, E4M3, "bhsd")
    a["vs"].fill_(2.0 ** power)
    a["ks"] *= 16.0  # logits of up to 60 or so: maxima move
    lengths = torch.randint(1, 1001, (12,), generator=torch.Generator().manual_seed(7), dtype=torch.int32).to(DEV)
    ref, size, top, biggest = formula(a, lengths, "bhsd")
    e = (D + 16) * 2.0 ** -24 * biggest
    bound = U[BF16] * ref.abs() + (2.0 ** -11 + 2 * e + 2.0 ** -20) * size + 2.0 ** -25 * 1000 * 448 * top + 2.0 ** -133
    off = (call(a, lengths, "bhsd").double() - ref).abs() / bound
    assert bool((off <= 1).all()), float(off.max())
