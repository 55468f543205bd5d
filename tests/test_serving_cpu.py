"""CPU: the operators around the attention refuse what they cannot run, with the wrapper's
kinds of error, before any device work; the rotary table holds the formula's angles."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import tilelang_fa2_4d_mask as api
from fa2_with_4d_mask_b200 import _lib


@pytest.mark.parametrize("base,dim", [(1e4, 128), (5e5, 96), (0.5, 20)])
def test_rotary_table(base, dim):
    rope = api.MultiAxisRotary(dim, (dim // 2 - 2, 0, 2), base=base)
    turns, axes = _lib.host().table_turns(rope._table)
    assert len(turns) == dim // 2 and axes == (0,) * (dim // 2 - 2) + (2, 2)
    for i in range(dim // 2):
        want = base ** (-2.0 * i / dim) / (2 * math.pi) % 1.0
        assert abs((turns[i] / 2.0 ** 64 - want + 0.5) % 1.0 - 0.5) < 2.0 ** -50


@pytest.mark.parametrize("args,kw,msg", [
    ((63, (31,)), {}, "head_dim must be even"),
    ((258, (129,)), {}, "head_dim must be even"),
    ((64, (31,)), {}, "sections must add up"),
    ((64, ()), {}, "sections must add up"),
    ((64, (40, -8)), {}, "sections must add up"),
    ((64, (32,)), dict(rotary_dim=66), "rotary_dim must be even"),
    ((64, (32,)), dict(pairing="third"), "unsupported pairing"),
    ((64, (32,)), dict(base=0.0), "base must be positive"),
    ((64, (32,)), dict(base=float("inf")), "base must be positive"),
])
def test_rotary_construction_refusals(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        api.MultiAxisRotary(*args, **kw)


def _new(B=2, H=2, T=3, D=64, dtype=torch.bfloat16):
    return torch.zeros(B, H, T, D, dtype=dtype)


POS = torch.zeros(1, 2, 3, dtype=torch.int64)


@pytest.mark.parametrize("q,k,pos,kw,msg", [
    (_new()[0], _new(), POS, {}, "query must be a rank-4"),
    (_new(dtype=torch.float32), _new(), POS, {}, "query must be fp16 or bf16"),
    (_new(), _new(dtype=torch.float16), POS, {}, "key must have the dtype"),
    (_new(), _new(B=1), POS, {}, "key must have the batch size"),
    (_new(), _new(T=4), POS, {}, "key must have the batch size"),
    (_new(), _new(D=32), POS, {}, "key has head dimension 32"),
    (_new(), _new(), POS[0], {}, "positions must be an integer tensor of shape"),
    (_new(), _new(), POS.expand(2, 2, 3), {}, "positions must be an integer tensor of shape"),
    (_new(), _new(), POS[..., :2], {}, "positions must be an integer tensor of shape"),
    (_new(), _new(), POS.float(), {}, "positions must be an integer tensor"),
    (_new(), _new(), POS, dict(layout="sbhd"), "unsupported layout"),
])
def test_rotary_refusals(q, k, pos, kw, msg):
    with pytest.raises(ValueError, match=msg):
        api.MultiAxisRotary(64, (32,))(q, k, pos, **kw)


def test_no_cpu_fallback():
    rope = api.MultiAxisRotary(64, (32,))
    with pytest.raises(RuntimeError, match="CUDA"):
        rope(_new(), _new(), POS)
    cache, n = _new(T=8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        rope.append(_new(), _new(), _new(), POS, cache, cache.clone(), n)
    with pytest.raises(RuntimeError, match="CUDA"):
        api.shared_prefix_attention(_new(), None, None, cache, cache, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        api.evict_by_weight(cache, cache, torch.zeros(2, 2, 8), n, keep=4)


@pytest.mark.parametrize("change,msg", [
    (dict(v=_new(H=1)), "value must have the heads of key"),
    (dict(kc=_new(T=8)[:1]), "key cache has shape"),
    (dict(vc=_new(T=9)), "value cache has shape"),
    (dict(vc=_new(T=8, dtype=torch.float16)), "value cache must be"),
    (dict(kc=_new(T=0), vc=_new(T=0)), "no slots"),
    (dict(n=torch.zeros(2)), "lengths must be"),
    (dict(n=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
    (dict(n=torch.zeros(4, dtype=torch.int32)[::2]), "lengths must be"),
    (dict(w=torch.zeros(2, 2, 7)), "weights must be"),
    (dict(w=torch.zeros(2, 8, 2).transpose(1, 2)), "weights must be"),
    (dict(w=torch.zeros(2, 2, 8, dtype=torch.float64)), "weights must be"),
    (dict(k=_new().requires_grad_()), "no gradient"),
    (dict(vc=_new(B=1, T=8).expand(2, -1, -1, -1)), "may not repeat memory"),
    (dict(w=torch.zeros(1, 2, 8).expand(2, -1, -1)), "may not repeat memory"),
    (dict(kc=_new(D=8, T=64).transpose(2, 3)), "expected batch|unit head-dim"),
    (dict(vc=torch.zeros(2, 2, 64, 8, dtype=torch.bfloat16).transpose(2, 3)), "unit head-dim"),
])
def test_append_refusals(change, msg):
    a = dict(q=_new(), k=_new(), v=_new(), kc=_new(T=8), vc=_new(T=8), n=torch.zeros(2, dtype=torch.int32), w=None)
    a.update(change)
    with pytest.raises(ValueError, match=msg):
        api.MultiAxisRotary(64, (32,)).append(a["q"], a["k"], a["v"], POS, a["kc"], a["vc"], a["n"], weights=a["w"])


PRE = torch.zeros(2, 5, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("change,msg", [
    (dict(q=_new()[0]), "query must be a rank-4"),
    (dict(q=_new(dtype=torch.float32)), "fp16 or bf16"),
    (dict(q=_new(H=3)), "divisible"),
    (dict(q=_new(D=80), k=_new(D=80), v=_new(D=80), pk=None, pv=None), "head dim 80 is not built"),
    (dict(k=_new()[0]), "key cache must be a rank-4"),
    (dict(v=_new(T=4)), "value cache has shape"),
    (dict(k=_new(B=1)), "key cache has shape"),
    (dict(pv=None), "go together"),
    (dict(pk=PRE[:1]), "prefix_key must have shape"),
    (dict(pv=PRE[:, :4]), "prefix_value must have shape"),
    (dict(pk=PRE.half()), "prefix_key must be"),
    (dict(n=torch.zeros(2, dtype=torch.int64)), "lengths must be"),
    (dict(mask=torch.ones(2, 2, 3, 4, dtype=torch.bool)), "mask must be a bool tensor"),
    (dict(mask=torch.ones(2, 2, 3, 3)), "mask must be a bool tensor"),
    (dict(mask=torch.ones(2, 3, 3, 3, dtype=torch.bool)), "mask must be a bool tensor"),
    (dict(weights=torch.zeros(2, 2, 4)), "weights must be"),
    (dict(weights=torch.zeros(2, 1, 3).expand(-1, 2, -1)), "may not repeat memory"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(layout="sbhd"), "unsupported layout"),
    (dict(q=_new().requires_grad_()), "no gradient"),
])
def test_shared_prefix_refusals(change, msg):
    a = dict(q=_new(), pk=PRE, pv=PRE, k=_new(), v=_new(), n=torch.zeros(2, dtype=torch.int32))
    kw = {x: change[x] for x in change if x not in a}
    a.update({x: change[x] for x in change if x in a})
    with pytest.raises(ValueError, match=msg):
        api.shared_prefix_attention(a["q"], a["pk"], a["pv"], a["k"], a["v"], a["n"], **kw)


@pytest.mark.parametrize("change,msg", [
    (dict(keep=0), "must fit in keep"),
    (dict(keep=5, sinks=3, recent=3), "must fit in keep"),
    (dict(sinks=-1), "must fit in keep"),
    (dict(key=_new(T=8).float()), "fp16 or bf16"),
    (dict(weights=None), "weights are required"),
    (dict(weights=torch.zeros(2, 2, 9)), "weights must be"),
    (dict(out=(_new(T=3), _new(T=3), torch.zeros(2, 2, 3))), "at least keep = 4"),
    (dict(out=(_new(T=4), _new(T=5), torch.zeros(2, 2, 4))), "value cache has shape"),
    (dict(out=(_new(H=1, T=4).expand(-1, 2, -1, -1), _new(T=4), torch.zeros(2, 2, 4))), "may not repeat memory"),
])
def test_evict_refusals(change, msg):
    a = dict(key=_new(T=8), value=_new(T=8), weights=torch.zeros(2, 2, 8), lengths=torch.zeros(2, dtype=torch.int32), keep=4)
    a.update(change)
    first = [a.pop(x) for x in ("key", "value", "weights", "lengths")]
    with pytest.raises((ValueError, RuntimeError), match=msg):
        api.evict_by_weight(*first, **a)


def test_c_entries_refuse_without_device_work():
    lib = _lib.load_library()
    for name in ("fa4d_rotary", "fa4d_rotary_append", "fa4d_prefix_attention", "fa4d_evict"):
        assert getattr(lib, name)(None, None) == _lib.FA4D_ERR_INVALID and lib.fa4d_last_error()
        # A structure of zeros has no pointers and no sizes.
        zeros = ctypes.create_string_buffer(4096)
        assert getattr(lib, name)(zeros, None) in (_lib.FA4D_ERR_INVALID, _lib.FA4D_ERR_UNSUPPORTED)
    lib.fa4d_prefix_attention_workspace.restype = ctypes.c_size_t
    ws = lib.fa4d_prefix_attention_workspace
    assert ws(2, 1, 8, 2, 128, 100, 50, 0) > 0
    assert ws(2, 1, 8, 2, 128, 100, 50, 1) > ws(2, 1, 8, 2, 128, 100, 50, 0)
    assert ws(2, 1, 8, 3, 128, 100, 50, 0) == 0 and ws(2, 1, 8, 2, 80, 100, 50, 0) == 0 and ws(0, 1, 8, 2, 64, 1, 1, 0) == 0
