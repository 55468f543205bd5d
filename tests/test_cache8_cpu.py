"""CPU: norms and 8-bit caches refuse what they cannot run before any device work; the restatements
of codes and scales agree with torch's conversions."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib
from oracle.cache8 import join_block, least_scale, nearest_code, norm_ref, norm_rotary_grads
from oracle.serving import rotary_ref

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def new(B=2, H=2, T=3, D=64, dtype=torch.bfloat16):
    return torch.zeros(B, H, T, D, dtype=dtype)


POS = torch.zeros(1, 2, 3, dtype=torch.int64)


def norm_call(q=None, k=None, wq=None, wk=None, **kw):
    w = torch.ones(64)
    return api.MultiAxisRotary(64, (32,))(q if q is not None else new(), k if k is not None else new(), POS,
                                          query_norm=w if wq is None else wq, key_norm=w if wk is None else wk, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(wq=torch.ones(63)), "query_norm must have 64 elements"),
    (dict(wk=torch.ones(1, 64)), "key_norm must be a rank-1"),
    (dict(wk=3), "key_norm must be a rank-1"),
    (dict(wq=torch.ones(64).double()), "both be fp32 or both"),
    (dict(wq=torch.ones(64).half()), "both be fp32 or both"),
    (dict(wq=torch.ones(64).bfloat16()), "both be fp32 or both"),
    (dict(wk=torch.ones(64).bfloat16()), "both be fp32 or both"),
    (dict(eps=0.0), "eps must be positive"),
    (dict(eps=-1.0), "eps must be positive"),
    (dict(eps=1e-60), "eps must be positive"),
    (dict(eps=float("nan")), "eps must be positive"),
    (dict(eps=float("inf")), "eps must be positive"),
    (dict(eps="small"), "eps must be a number"),
    (dict(q=new(dtype=torch.float32)), "query must be fp16 or bf16"),
    (dict(k=new(D=32)), "key has head dimension 32"),
    (dict(layout="sbhd"), "unsupported layout"),
])
def test_norm_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        norm_call(**kw)


def test_norms_go_together():
    rope, w = api.MultiAxisRotary(64, (32,)), torch.ones(64)
    for kw in (dict(query_norm=w), dict(key_norm=w)):
        with pytest.raises(ValueError, match="go together"):
            rope(new(), new(), POS, **kw)
        with pytest.raises(ValueError, match="go together"):
            rope.append(new(), new(), new(), POS, new(T=8), new(T=8), torch.zeros(2, dtype=torch.int32), **kw)


def args8(code=E4M3, C=70, D=64):
    return dict(q=new(D=D), k=new(D=D), v=new(D=D), kc=new(T=C, D=D, dtype=code), vc=new(T=C, D=D, dtype=code),
                ks=torch.ones(2, 2, -(-C // 64)), vs=torch.ones(2, 2, -(-C // 64)), n=torch.zeros(2, dtype=torch.int32))


def append8(a, **kw):
    D = a["q"].shape[3]
    return api.MultiAxisRotary(D, (D // 2,)).append(a["q"], a["k"], a["v"], POS, a["kc"], a["vc"], a["n"], key_scale=a["ks"],
                                                    value_scale=a["vs"], **kw)


def attend8(a, **kw):
    return api.shared_prefix_attention(a["q"], None, None, a["kc"], a["vc"], a["n"], key_scale=a["ks"], value_scale=a["vs"], **kw)


BOTH = [
    (dict(kc=new(T=70)), "must be float8_e4m3fn or int8"),
    (dict(vc=new(T=70, dtype=INT8)), "must be float8_e4m3fn or int8, as the other"),
    (dict(vc=new(T=71, dtype=E4M3)), "value cache has shape"),
    (dict(kc=new(T=0, dtype=E4M3), vc=new(T=0, dtype=E4M3)), "no slots"),
    (dict(ks=torch.ones(2, 2, 1)), "key_scale must be an fp32 tensor of shape \\[2, 2, 2\\]"),
    (dict(vs=torch.ones(2, 2, 2).half()), "value_scale must be an fp32"),
    (dict(vs=torch.ones(2, 2, 2).transpose(1, 2)), "unit block stride"),
    (dict(vs=None), "go together"),
    (dict(ks=None), "go together"),
    (dict(ks=3), "must be fp32 tensors"),
    (dict(n=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
    (dict(q=new().requires_grad_()), "no gradient"),
    (dict(ks=torch.ones(2, 2, 2, requires_grad=True)), "no gradient"),
]


@pytest.mark.parametrize("change,msg", BOTH)
@pytest.mark.parametrize("call", [append8, attend8])
def test_refusals_of_8_bit_caches(call, change, msg):
    with pytest.raises(ValueError, match=msg):
        call({**args8(), **change})


@pytest.mark.parametrize("change,kw,msg", [
    ({}, dict(weights=torch.zeros(2, 2, 70)), "weights go with 16-bit"),
    (dict(kc=new(B=1, T=70, dtype=E4M3).expand(2, -1, -1, -1)), {}, "may not repeat memory"),
    (dict(vs=torch.ones(1, 2, 2).expand(2, -1, -1)), {}, "may not repeat memory"),
    (dict(kc=torch.zeros(2, 2, 70, 72, dtype=torch.int8)[..., :64].view(E4M3)), {}, "16-byte boundaries"),
    (dict(kc=torch.zeros(2, 2, 70, 80, dtype=torch.int8)[..., 3:67].view(E4M3)), {}, "16-byte boundaries"),
])
def test_append_refusals_of_8_bit_caches(change, kw, msg):
    with pytest.raises(ValueError, match=msg):
        append8({**args8(), **change}, **kw)


def test_append_needs_caches_of_their_own_and_whole_rows():
    a = args8()
    with pytest.raises(ValueError, match="of their own"):
        append8({**a, "vc": a["kc"]})
    with pytest.raises(ValueError, match="of their own"):
        append8({**a, "vs": a["ks"]})
    with pytest.raises(ValueError, match="multiple of 16"):
        append8(args8(D=72))
    turned = new(T=64, D=70, dtype=E4M3).transpose(2, 3)
    with pytest.raises(ValueError, match="unit head-dim"):
        append8({**a, "kc": turned})


@pytest.mark.parametrize("kw,msg", [
    (dict(weights=torch.zeros(2, 2, 70)), "weights go with 16-bit"),
    (dict(mask=torch.ones(2, 2, 3, 69, dtype=torch.bool)), "mask must be a bool tensor"),
    (dict(scale=float("nan")), "scale must be finite"),
])
def test_attention_refusals_of_8_bit_caches(kw, msg):
    with pytest.raises(ValueError, match=msg):
        attend8(args8(), **kw)
    with pytest.raises(ValueError, match="head dim 80 is not built"):
        attend8(args8(D=80))
    with pytest.raises(ValueError, match="key cache must be torch.bfloat16"):  # codes without scales
        api.shared_prefix_attention(new(), None, None, new(T=70, dtype=E4M3), new(T=70, dtype=E4M3), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("change,kw,msg", [
    (dict(x=new(T=70)), {}, "float8_e4m3fn or int8"),
    (dict(x=new(T=70, dtype=E4M3)[0]), {}, "cache must be a rank-4"),
    (dict(x=new(T=70, D=72, dtype=E4M3)), {}, "multiple of 16"),
    (dict(s=torch.ones(2, 2, 3)), {}, "scale must be an fp32 tensor of shape"),
    (dict(n=torch.zeros(2)), {}, "lengths must be"),
    ({}, dict(dtype=torch.float32), "dtype must be"),
    ({}, dict(dtype="bf16"), "dtype must be"),
    ({}, dict(layout="sbhd"), "unsupported layout"),
    (dict(s=torch.ones(2, 2, 2, requires_grad=True)), {}, "no gradient"),
])
def test_cache_values_refusals(change, kw, msg):
    a = {**dict(x=new(T=70, dtype=INT8), s=torch.ones(2, 2, 2), n=torch.zeros(2, dtype=torch.int32)), **change}
    with pytest.raises(ValueError, match=msg):
        api.cache_values(a["x"], a["s"], a["n"], **kw)


def test_no_cpu_fallback():
    for code in (E4M3, INT8):
        a = args8(code)
        for call in (lambda: append8(a), lambda: attend8(a), lambda: api.cache_values(a["kc"], a["ks"], a["n"]), norm_call):
            with pytest.raises(RuntimeError, match="CUDA"):
                call()


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(grad_mode):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        w, a = torch.ones(64), args8()
        for call in (lambda: norm_call(q=dual(new())), lambda: norm_call(wk=dual(w)), lambda: append8({**a, "k": dual(new())}),
                     lambda: append8({**a, "vs": dual(a["vs"])}), lambda: append8(a, query_norm=w, key_norm=dual(w)),
                     lambda: attend8({**a, "q": dual(new())}), lambda: attend8({**a, "ks": dual(a["ks"])}),
                     lambda: api.cache_values(a["kc"], dual(a["ks"]), a["n"])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_c_entries_refuse_without_device_work():
    lib = _lib.load_library()
    for name in ("fa4d_norm_rotary", "fa4d_norm_rotary_bwd", "fa4d_norm_append", "fa4d_cache_values", "fa4d_prefix_attention_8bit"):
        assert getattr(lib, name)(None, None) == _lib.FA4D_ERR_INVALID and lib.fa4d_last_error()
        zeros = ctypes.create_string_buffer(8192)
        assert getattr(lib, name)(zeros, None) in (_lib.FA4D_ERR_INVALID, _lib.FA4D_ERR_UNSUPPORTED)
    ws = lib.fa4d_prefix_attention_8bit_workspace
    ws.restype = ctypes.c_size_t
    assert ws(2, 1, 8, 2, 128, 100, 50) > ws(2, 1, 8, 2, 128, 0, 50) > 0
    assert ws(2, 1, 8, 3, 128, 0, 50) == 0 and ws(2, 1, 8, 2, 80, 0, 50) == 0 and ws(0, 1, 8, 2, 64, 1, 1) == 0
    ws = lib.fa4d_norm_rotary_bwd_workspace
    ws.restype = ctypes.c_size_t
    assert ws(2, 100, 8, 2, 128) > 0 and ws(0, 1, 8, 2, 128) == 0 and ws(1, 1, 8, 2, 258) == 0


def test_codes_round_as_torch_converts():
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).to(torch.float64)
    every = every[torch.isfinite(every)]
    x = torch.cat([every, (every[1:] + every[:-1]) / 2, torch.randn(2000, dtype=torch.float64) * 100])
    x = x.clamp(-448, 448)
    assert torch.equal(nearest_code(x, E4M3).abs(), x.float().to(E4M3).double().abs())
    assert torch.equal(nearest_code(torch.tensor([0.5, 1.5, -2.5, 126.6], dtype=torch.float64), INT8),
                       torch.tensor([0.0, 2.0, -2.0, 127.0], dtype=torch.float64))


@pytest.mark.parametrize("code,top", [(E4M3, 448.0), (INT8, 127.0)])
def test_scales_are_the_least_powers_of_two(code, top):
    for e in (-130, -126, -3, 0, 17):
        for f in (1.0, 1.0 + 2.0 ** -23, 0.51, 0.5):
            s = least_scale(top * f * 2.0 ** e, code)
            assert math.log2(s) == int(math.log2(s)) >= -126
            assert top * f * 2.0 ** e <= top * s and (s == 2.0 ** -126 or top * f * 2.0 ** e > top * s / 2)
    assert least_scale(0.0, code) == 2.0 ** -126 and math.isnan(least_scale(math.inf, code))
    old = torch.full((2, 4), top)
    codes, s = join_block(old, 1.0, torch.full((1, 4), 4 * top, dtype=torch.float64), 2, code)
    assert s == 4.0 and torch.equal(codes[2], torch.full((4,), top, dtype=torch.float64))


def test_the_gradient_formula_matches_autograd():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 5, 8, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(8, generator=g, dtype=torch.float64, requires_grad=True)
    dy, pos = torch.randn(2, 3, 5, 8, generator=g, dtype=torch.float64), torch.randint(0, 99, (1, 2, 5), generator=g)
    y = rotary_ref(norm_ref(x, w, 1e-3), pos, (4,), base=1e4)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    _, dx, dw = norm_rotary_grads(x.detach(), w.detach(), dy, pos, (4,), eps=1e-3, base=1e4)
    assert torch.allclose(gx, dx, rtol=1e-12, atol=1e-13) and torch.allclose(gw, dw, rtol=1e-12, atol=1e-13)
