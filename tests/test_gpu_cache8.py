"""Caches in 8 bits: appending (norm, turn, scale, codes, earlier codes anew) and reading back.

Values joins as they are: its codes and scales are equal to the plain form's.  Keys are turned (and
normalised) in 32 bits first, off by ((D + 16) 2^-24 + 2^-20) max|n| at most (as without a cache),
and rounded to the nearest code: 2^-4 of the value or, of e4m3's least exponent, 2^-10 of the scale;
half a scale in int8.  Key scales are equal where that error does not reach the border of a power of
two, as here (asserted)."""

from __future__ import annotations

import math

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import BLOCK, LARGEST, join_block, least_scale, norm_ref, values_ref
from oracle.serving import rotary_ref

DEV = torch.device("cuda", 0)
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16


def randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def swap(x, layout):
    """Between a layout and the canonical [B, H, T, D]."""
    return x if layout == "bhsd" else x.transpose(1, 2)


def cache(g, B, Hk, C, D, code, layout):
    """Random codes (of all kinds but NaN) and powers of two."""
    if code == INT8:
        c = torch.randint(-127, 128, (B, Hk, C, D), generator=g).to(torch.int8)
    else:
        c = (torch.randn(B, Hk, C, D, generator=g) * 100).clamp(-448, 448).to(E4M3)
    c = c.to(DEV)
    c = c if layout == "bhsd" else c.view(torch.uint8).transpose(1, 2).contiguous().view(code)
    return c, torch.exp2(torch.randint(-7, -4, (B, Hk, -(-C // BLOCK)), generator=g).float()).to(DEV)


def canonical(x, layout):
    """Codes as values in 64 bits."""
    return swap(x.to(torch.float64), layout)


def check_append(rope, q, k, v, pos, kc, vc, ks, vs, lengths, sections, layout, weights=None, eps=1e-6, base=1e4, exact=False, **kw):
    """`exact`: the turn is by no angle, so that keys are exact and may lie at borders."""
    code, B, D = kc.dtype, q.shape[0], q.shape[3]
    C, T, Hk = swap(kc, layout).shape[2], swap(k, layout).shape[2], swap(k, layout).shape[1]
    before = [canonical(kc, layout).clone(), canonical(vc, layout).clone(), ks.clone(), vs.clone()]
    bits = [swap(x.view(torch.uint8), layout).clone() for x in (kc, vc)]
    norms = {} if weights is None else dict(query_norm=weights[0], key_norm=weights[1], eps=eps)
    got_q, new = rope.append(q, k, v, pos, kc, vc, lengths, key_scale=ks, value_scale=vs, layout=layout, **norms)
    had = lengths.clamp(min=0)
    assert torch.equal(new, (had + T).clamp(max=C))
    plain_q, _ = rope(q, k, pos, layout=layout, **norms)
    assert float((got_q.double() - plain_q.double()).abs().max()) <= 2 * torch.finfo(q.dtype).eps * float(plain_q.abs().max())
    nk = k.double() if weights is None else norm_ref(k, weights[1], eps)
    xk, xv = swap(rotary_ref(nk, pos, sections, base=base, layout=layout, **kw), layout), swap(v.double(), layout)
    err = ((D + 16) * 2.0 ** -24 + 2.0 ** -20) * float(nk[torch.isfinite(nk)].abs().max())
    out_k, out_v = canonical(kc, layout), canonical(vc, layout)
    now = [swap(x.view(torch.uint8), layout) for x in (kc, vc)]
    for b in range(B):
        n = int(had[b])
        end = min(n + T, C)
        for j in range(-(-C // BLOCK)):
            lo, hi = j * BLOCK, min((j + 1) * BLOCK, C)
            first, last = max(lo, n), min(hi, end)
            if first >= last:  # untouched, stale slots too
                for h in range(Hk):
                    for i in range(2):
                        assert torch.equal(now[i][b, h, lo:hi], bits[i][b, h, lo:hi])
                for s, was in ((ks, before[2]), (vs, before[3])):
                    assert torch.equal(s.view(torch.int32)[b, :, j], was.view(torch.int32)[b, :, j])
                continue
            for h in range(Hk):
                # values: exactly
                want, scale = join_block(before[1][b, h, lo:last], float(before[3][b, h, j]), xv[b, h, first - n:last - n],
                                         first - lo, code)
                assert float(vs[b, h, j]) == scale or (math.isnan(scale) and math.isnan(float(vs[b, h, j])))
                assert torch.equal(out_v[b, h, lo:last], want)
                # keys: scale, earlier codes, new codes
                fresh, old = xk[b, h, first - n:last - n], float(before[2][b, h, j])
                if not torch.isfinite(fresh).all():
                    assert math.isnan(float(ks[b, h, j]))
                    continue
                want, scale = join_block(before[0][b, h, lo:last], old, fresh, first - lo, code)
                most = float(fresh.abs().max())
                assert exact or least_scale(most * (1 - 1e-5), code) == least_scale(most * (1 + 1e-5), code), "a border: choose another seed"
                assert float(ks[b, h, j]) == scale or (math.isnan(scale) and math.isnan(float(ks[b, h, j])))
                assert torch.equal(out_k[b, h, lo:first], want[:first - lo])
                if math.isnan(scale):
                    continue
                got = out_k[b, h, first:last] * scale
                half = scale / 2 if code == INT8 else torch.maximum(2.0 ** -4 * fresh.abs(), torch.tensor(2.0 ** -10 * scale, device=DEV))
                assert bool(((got - fresh).abs() <= half + err).all())
            # behind the last token: as it was
            for i in range(2):
                assert torch.equal(now[i][b, :, last:hi], bits[i][b, :, last:hi])
    for x, s in ((kc, ks), (vc, vs)):
        for dtype in (BF16, FP16):
            values = api.cache_values(x, s, new, dtype=dtype, layout=layout)
            ref = values_ref(swap(x, layout), s, new)
            assert torch.equal(swap(values, layout).nan_to_num(9.0), ref.to(dtype).nan_to_num(9.0))
            # bf16 holds every value, but for 2^128, to which its largest (255 codes of 2^120) is rounded.
            inside = ref.abs() < 2.0 ** 128
            assert dtype == FP16 or torch.equal(swap(values, layout).double()[inside], ref[inside])


CASES = [
    # (B, T, Hq, Hk, D, rotary_dim, sections, pairing, dtype, C, code, layout, normed)
    (1, 1, 1, 1, 64, None, (32,), "half", BF16, 1, E4M3, "bhsd", False),
    (3, 1, 4, 2, 128, None, (16, 24, 24), "half", BF16, 200, E4M3, "bshd", True),
    (3, 1, 4, 2, 128, None, (16, 24, 24), "half", BF16, 200, INT8, "bshd", True),
    (2, 7, 3, 3, 96, 64, (32,), "adjacent", FP16, 100, E4M3, "bhsd", True),
    (2, 63, 4, 1, 64, None, (8, 24), "adjacent", FP16, 129, INT8, "bshd", False),
    (1, 64, 2, 2, 256, 96, (48,), "half", BF16, 130, E4M3, "bshd", True),
    (1, 65, 2, 2, 256, None, (128,), "adjacent", FP16, 321, INT8, "bhsd", True),
    (2, 200, 8, 2, 128, None, (64,), "half", BF16, 500, E4M3, "bhsd", False),
    (2, 131, 2, 1, 80, 36, (9, 9), "half", BF16, 200, INT8, "bshd", True),  # no runs of 8
    (2, 33, 2, 1, 16, 6, (3,), "adjacent", FP16, 64, E4M3, "bhsd", False),
    (70, 2, 2, 3, 64, None, (32,), "half", BF16, 70, E4M3, "bshd", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,rot,sections,pairing,dtype,C,code,layout,normed", CASES)
def test_append_and_read_back(B, T, Hq, Hk, D, rot, sections, pairing, dtype, C, code, layout, normed):
    g = torch.Generator().manual_seed(B * 1000 + T)
    rope = api.MultiAxisRotary(D, sections, base=1e4, rotary_dim=rot, pairing=pairing)
    shape = lambda H: (B, H, T, D) if layout == "bhsd" else (B, T, H, D)  # noqa: E731
    q, k, v = randn(g, shape(Hq), dtype), randn(g, shape(Hk), dtype), randn(g, shape(Hk), dtype, 2.0)
    pos = torch.randint(-50, 9999, (len(sections), B, T), generator=g, dtype=torch.int32).to(DEV)
    (kc, ks), (vc, vs) = cache(g, B, Hk, C, D, code, layout), cache(g, B, Hk, C, D, code, layout)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(DEV) for _ in range(2)] if normed else None
    lengths = torch.randint(0, C - T + 1, (B,), generator=g, dtype=torch.int32)
    lengths[0] = min(C - T, 60)
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, lengths.to(DEV), sections, layout, weights=w, base=1e4, rotary_dim=rot,
                 pairing=pairing)
    assert _lib.device_status(DEV) == 0


def plain(g, B=2, T=3, Hk=2, D=64, C=150, code=E4M3, dtype=BF16):
    rope = api.MultiAxisRotary(D, (D // 2,))
    q, k, v = (randn(g, (B, Hk, T, D), dtype) for _ in range(3))
    (kc, ks), (vc, vs) = cache(g, B, Hk, C, D, code, "bhsd"), cache(g, B, Hk, C, D, code, "bhsd")
    pos = torch.arange(T, device=DEV).expand(1, B, T)
    return rope, [q, k, v, pos, kc, vc, ks, vs]


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_token_by_token_equals_the_prompt_for_growing_magnitudes(code):
    """80 tokens one by one, each block's largest last, and from small to large: scales are the
    prompt's; codes were rounded anew at most a few times: each time by at most half a code of then,
    at most one code of the last scale in all (1/2 + 1/4 + ...)."""
    g = torch.Generator().manual_seed(4)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, T=80, code=code)
    grow = torch.exp2(torch.arange(80, device=DEV) / 8.0)[:, None]
    k, v = (k.float() * grow).to(BF16), (v.float() * grow).to(BF16)
    one = [x.clone() for x in (kc, vc, ks, vs)]
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, n, (32,), "bhsd")
    for t in range(80):
        _, n = rope.append(q[:, :, t:t + 1], k[:, :, t:t + 1], v[:, :, t:t + 1], pos[:, :, t:t + 1], one[0], one[1], n,
                           key_scale=one[2], value_scale=one[3])
    assert n.tolist() == [80, 80] and torch.equal(one[2], ks) and torch.equal(one[3], vs)
    for a, b, s in ((one[0], kc, ks), (one[1], vc, vs)):
        x, y = (api.cache_values(i, s, n).double()[:, :, :80] for i in (a, b))
        step = s.double().repeat_interleave(BLOCK, 2)[:, :, :80, None]
        # e4m3: only codes that fall below its least normal step are rounded anew, to 2^-9.
        bound = 1.5 * step if code == INT8 else torch.maximum(2.0 ** -9 * step * 1.5, torch.zeros_like(x))
        assert bool(((x - y).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scales_at_their_borders(code):
    """Magnitudes at, just above and far from the largest code times a power of two; zeros; bf16's
    least and largest."""
    g = torch.Generator().manual_seed(8)
    top = LARGEST[code]
    some = [0.0, top, -top * 2 ** -9, top * 2 ** 20, 1.0, 2.0 ** -133, -3.3895e38, 1e-38, 2.0 ** -126]
    above = torch.tensor([top, top * 2 ** -30], dtype=BF16).view(torch.int16) + 1  # the next bf16
    some += above.view(BF16).tolist()
    rope, (_, _, _, _, kc, vc, ks, vs) = plain(g, B=len(some), T=1, code=code)
    x = torch.zeros(len(some), 2, 1, 64, dtype=BF16, device=DEV)
    x[:, :, 0, 3] = torch.tensor(some, device=DEV)[:, None].to(BF16)
    n = torch.zeros(len(some), dtype=torch.int32, device=DEV)
    check_append(rope, x, x, x, torch.zeros(1, 1, 1, dtype=torch.int64, device=DEV), kc, vc, ks, vs, n, (32,), "bhsd",
                 exact=True)
    want = [least_scale(abs(float(y)), code) for y in x[:, 0, 0, 3]]
    assert ks[:, 0, 0].tolist() == want and vs[:, 1, 0].tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_infinities_and_nan_make_their_block_nan_until_it_starts_anew(code):
    g = torch.Generator().manual_seed(9)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, T=70, code=code)
    k[0, 0, 3, 5], v[1, 1, 66, 2] = float("nan"), -float("inf")
    n = torch.tensor([0, 10], dtype=torch.int32, device=DEV)
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, n, (32,), "bhsd")
    new = n + 70
    bad_k, bad_v = (torch.isnan(api.cache_values(c, s, new)) for c, s in ((kc, ks), (vc, vs)))
    assert bad_k[0, 0, :64].all() and not bad_k[0, 0, 64:].any() and not bad_k[1].any() and not bad_k[0, 1].any()
    assert bad_v[1, 1, 64:80].all() and not bad_v[1, 1, :64].any() and not bad_v[0].any()
    # A finite token behind them leaves it so; one that starts the block anew does not.
    one = [x[:, :, :1].contiguous() for x in (q, v.nan_to_num(0.0), v.nan_to_num(0.0))]
    for lengths, nan in ((5, True), (0, False)):
        check_append(rope, *one, pos[:, :, :1], kc, vc, ks, vs, torch.tensor([lengths, 0], dtype=torch.int32, device=DEV), (32,), "bhsd")
        assert math.isnan(float(ks[0, 0, 0])) == nan


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_squares_beyond_32_bits_become_rows_of_zeros(code):
    """Finite tokens whose sum of squares is infinite in 32 bits: r = 0, as in a plain norm in 32
    bits; their neighbours in the block keep a finite scale."""
    g = torch.Generator().manual_seed(10)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, T=5, code=code)
    k[0, 1, 2] = 1e30
    k[1, 0, :, 7] = -3e38
    n = torch.tensor([0, 63], dtype=torch.int32, device=DEV)
    w = torch.ones(64, device=DEV)
    rope.append(q, k, v, pos, kc, vc, n, key_scale=ks, value_scale=vs, query_norm=w, key_norm=w)
    got = [api.cache_values(kc, ks, n + 5)[b, :, n[b]:n[b] + 5].float() for b in range(2)]
    assert all(bool(torch.isfinite(x).all()) for x in got)
    assert not got[0][1, 2].any() and not got[1][0].any()
    for x in (got[0][0], got[0][1, 3], got[1][1]):
        assert bool((x != 0).any(-1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_full_and_odd_lengths(code):
    """Tokens past the capacity are dropped and count for nothing, in a block that ends there too."""
    g = torch.Generator().manual_seed(10)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, B=6, T=9, C=70, code=code)
    v[:, :, 5:] *= 1000
    n = torch.tensor([65, 70, 61, -3, 1000, 64], dtype=torch.int32, device=DEV)
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, n, (32,), "bhsd")
    assert _lib.device_status(DEV) == _lib.DEV_CACHE_FULL and _lib.device_status(DEV) == 0
    got = api.cache_values(kc, ks, n)
    assert not got[3].any() and got[4].any()


@pytest.mark.gpu
def test_caches_and_tokens_with_strides_of_their_own():
    """A cache within a wider one, scales within others, tokens off 16-byte boundaries."""
    g = torch.Generator().manual_seed(11)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, T=5)
    n = torch.tensor([62, 3], dtype=torch.int32, device=DEV)
    wide = torch.zeros(2, 3, 2, 150, 96, dtype=torch.uint8, device=DEV)
    kw, vw = (wide[:, i, :, :, 16:80].view(E4M3) for i in (0, 2))
    kw.view(torch.uint8).copy_(kc.view(torch.uint8)), vw.view(torch.uint8).copy_(vc.view(torch.uint8))
    scales = torch.zeros(2, 2, 9, device=DEV)
    ksw, vsw = scales[..., 1:4], scales[..., 5:8]
    ksw.copy_(ks), vsw.copy_(vs)
    pad = torch.empty(k.numel() + 3, dtype=BF16, device=DEV)
    odd = pad[3:].view(k.shape)
    odd.copy_(k)
    check_append(rope, q, odd, v.transpose(2, 3).contiguous().transpose(2, 3), pos, kw, vw, ksw, vsw, n, (32,), "bhsd")
    check_append(rope, q, k, v, pos, kc, vc, ks, vs, n, (32,), "bhsd")
    assert torch.equal(kw.view(torch.uint8), kc.view(torch.uint8)) and torch.equal(vsw, vs)
    assert not wide[:, 1].any() and not wide[..., :16].any() and not wide[..., 80:].any()
    # Reading back a cache off 16-byte boundaries copies it first.
    off = torch.zeros(2, 2, 150, 65, dtype=torch.uint8, device=DEV)[..., 1:]
    off.copy_(kc.view(torch.uint8))
    assert torch.equal(api.cache_values(off.view(E4M3), ks, n), api.cache_values(kc, ks, n))


@pytest.mark.gpu
def test_empty_other_stream_and_graph():
    g = torch.Generator().manual_seed(12)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g)
    n = torch.tensor([5, 70], dtype=torch.int32, device=DEV)
    none, new = rope.append(q[:, :, :0], k[:, :, :0], v[:, :, :0], pos[:, :, :0], kc, vc, n, key_scale=ks, value_scale=vs)
    assert none.shape[2] == 0 and torch.equal(new, n)
    assert api.cache_values(kc[:0], ks[:0], n[:0]).shape == kc[:0].shape
    start = [x.clone() for x in (kc, vc, ks, vs)]

    def step(caches, n):
        kc, vc, ks, vs = caches
        q2, new = rope.append(q, k, v, pos, kc, vc, n, key_scale=ks, value_scale=vs)
        return q2, new, api.cache_values(kc, ks, new), api.cache_values(vc, vs, new)

    want = step([kc, vc, ks, vs], n)
    want2 = step([kc, vc, ks, vs], want[1])
    side, mine = torch.cuda.Stream(), [x.clone() for x in start]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(mine, n * 1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    mine, static = [x.clone() for x in start], n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(mine, static)
        static.copy_(got[1])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got[2:], want[2:]))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want2)) and torch.equal(static, want2[1])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The last request's codes lie past 2^32 bytes."""
    g = torch.Generator().manual_seed(13)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g, C=70)
    store = torch.zeros(2 ** 32 + 2 * 70 * 64 + 64, dtype=torch.uint8, device=DEV)
    big = store.as_strided((2, 2, 70, 64), (2 ** 32 + 64, 70 * 64, 64, 1)).view(E4M3)
    big.view(torch.uint8).copy_(kc.view(torch.uint8))
    n = torch.tensor([5, 62], dtype=torch.int32, device=DEV)
    check_append(rope, q, k, v, pos, big, vc, ks.clone(), vs.clone(), n, (32,), "bhsd")


@pytest.mark.gpu
def test_autograd_sees_the_writes():
    g = torch.Generator().manual_seed(14)
    rope, (q, k, v, pos, kc, vc, ks, vs) = plain(g)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    before = [x._version for x in (kc, vc, ks, vs)]
    rope.append(q, k, v, pos, kc, vc, n, key_scale=ks, value_scale=vs)
    assert all(x._version > b for x, b in zip((kc, vc, ks, vs), before))
    with torch.inference_mode():
        rope.append(q, k, v, pos, kc * 1 if kc.dtype == INT8 else kc.clone(), vc.clone(), n, key_scale=ks.clone(), value_scale=vs.clone())
