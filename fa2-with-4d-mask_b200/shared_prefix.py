"""Serving: attention of a batch's new tokens over a prefix that all requests share and each
request's own cache, and eviction from the caches by the attention weight their entries
received.

A decode step rotates and appends the new tokens (``MultiAxisRotary.append``), attends
(``shared_prefix_attention``, which can accumulate ``weights``) and, when caches run full,
shrinks them (``evict_by_weight``).  Everything is enqueued on the current stream without a
host synchronisation, so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .rotary import Layout, _bth, check_cache


def _no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """x with rows that 16-byte accesses can reach: itself, or a copy."""
    s = x.stride()
    ok = s[-1] == 1 and x.data_ptr() % 16 == 0 and all(n % 8 == 0 for n in s[:-1])
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def shared_prefix_attention(
    query: torch.Tensor,
    prefix_key: Optional[torch.Tensor],
    prefix_value: Optional[torch.Tensor],
    key: torch.Tensor,
    value: torch.Tensor,
    lengths: torch.Tensor,
    *,
    mask: Optional[torch.Tensor] = None,
    weights: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    is_causal: bool = True,
    layout: Layout = "bhsd",
) -> torch.Tensor:
    """Softmax attention of T new tokens per request over the shared prefix and the request's
    own cache together; the prefix is read once for the whole batch.

    Args:
        query: fp16/bf16 ``[B, Hq, T, D]`` ("bhsd") or ``[B, T, Hq, D]`` ("bshd"), head dim
            64, 96, 128 or 256; meant for few tokens (a decode step, a draft's verification).
        prefix_key/prefix_value: ``[Hk, P, D]`` or ``[P, Hk, D]``; None for no prefix.
        key/value: the caches, ``[B, Hk, C, D]`` or ``[B, C, Hk, D]``, ``Hq % Hk == 0``; what
            lies past a request's length is never used.
        lengths: int32 ``[B]``, entries of each cache, the T new tokens included.
        mask: optional bool ``[B or 1, Hq or 1, T, C]`` over the own cache, True keeps.
        weights: optional fp32 ``[B, Hk, C]``; gains in place the probability each own entry
            received, summed over the group's query heads and the T tokens.
        scale: softmax scale, ``head_dim ** -0.5`` by default.
        is_causal: new token t sees the own entries up to its own, ``lengths - T + t``.

    Returns:
        The output in the query's layout; rows that see no key are 0.

    Rows that are not on 16-byte boundaries are copied first.  There is no gradient.
    """
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"unsupported layout: {layout}")
    if not isinstance(query, torch.Tensor) or query.dim() != 4:
        raise ValueError("query must be a rank-4 tensor")
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"query must be fp16 or bf16, got {query.dtype}")
    if not isinstance(key, torch.Tensor) or key.dim() != 4:
        raise ValueError("key cache must be a rank-4 tensor")
    if layout == "bhsd":
        B, Hq, T, D = query.shape
        Hk = key.shape[1]
    else:
        B, T, Hq, D = query.shape
        Hk = key.shape[2]
    if Hk == 0 or Hq % Hk != 0:
        raise ValueError(f"query heads ({Hq}) must be divisible by key/value heads ({Hk})")
    if D not in (64, 96, 128, 256):
        raise ValueError(f"head dim {D} is not built (64, 96, 128, 256)")
    C = check_cache(key, value, lengths, weights, layout, B, Hk, D, query)
    if (prefix_key is None) != (prefix_value is None):
        raise ValueError("prefix_key and prefix_value go together")
    P = 0
    if prefix_key is not None:
        seq = 1 if layout == "bhsd" else 0
        for name, x in (("prefix_key", prefix_key), ("prefix_value", prefix_value)):
            if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.shape[1 - seq] != Hk or x.shape[2] != D \
                    or x.shape != prefix_key.shape:
                raise ValueError(f"{name} must have shape " + (f"[{Hk}, P, {D}]" if seq else f"[P, {Hk}, {D}]"))
            if x.dtype != query.dtype or x.device != query.device:
                raise ValueError(f"{name} must be {query.dtype} on {query.device}")
        P = prefix_key.shape[seq]
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dim() != 4 or mask.dtype != torch.bool \
                or mask.shape[0] not in (1, B) or mask.shape[1] not in (1, Hq) or tuple(mask.shape[2:]) != (T, C):
            raise ValueError(f"mask must be a bool tensor of shape [{B} or 1, {Hq} or 1, {T}, {C}]")
        if mask.device != query.device:
            raise ValueError(f"mask must be on {query.device}, got {mask.device}")
        if mask.stride(3) != 1:
            mask = mask.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    _no_grad("shared_prefix_attention", query, prefix_key, prefix_value, key, value)
    if not query.is_cuda:
        raise RuntimeError("shared_prefix_attention runs on CUDA (sm_100a) tensors only")
    query, key, value = _rows16(query), _rows16(key), _rows16(value)
    out = torch.empty_like(query)
    if out.numel() == 0:
        return out
    pk_ptr = pv_ptr = None
    pk_stride = pv_stride = (0, 0)
    if P:
        # The prefix also goes through tensor maps, which have no stride of 0.
        prefix_key, prefix_value = (
            _rows16(x if all(s > 0 or n == 1 for s, n in zip(x.stride(), x.shape)) else x.contiguous())
            for x in (prefix_key, prefix_value))
        pk_ptr, pv_ptr = prefix_key.data_ptr(), prefix_value.data_ptr()
        s, z = prefix_key.stride(), prefix_value.stride()
        pk_stride, pv_stride = ((s[1], s[0]), (z[1], z[0])) if layout == "bhsd" else (s[:2], z[:2])
    device = query.device
    ws_bytes = _lib.prefix_attention_workspace(device.index, B, T, Hq, Hk, D, P, C, weights is not None)
    workspace = torch.empty((ws_bytes,), dtype=torch.uint8, device=device)
    args = _lib.PrefixAttentionArgs(
        query.data_ptr(), pk_ptr, pv_ptr, key.data_ptr(), value.data_ptr(), out.data_ptr(), lengths.data_ptr(),
        None if mask is None else mask.data_ptr(), None if weights is None else weights.data_ptr(),
        workspace.data_ptr(), ws_bytes, _bth(query, layout), pk_stride, pv_stride, _bth(key, layout),
        _bth(value, layout), _bth(out, layout), (0, 0, 0) if mask is None else _lib._bias_strides(mask),
        (0, 0) if weights is None else weights.stride()[:2], B, T, Hq, Hk, D, P, C, _lib._dtype_code(query.dtype),
        1 if is_causal else 0, scale)
    _lib.launch("fa4d_prefix_attention", args, device)
    return out


def evict_by_weight(
    key: torch.Tensor,
    value: torch.Tensor,
    weights: torch.Tensor,
    lengths: torch.Tensor,
    *,
    keep: int,
    sinks: int = 0,
    recent: int = 0,
    out: Optional[tuple] = None,
    layout: Layout = "bhsd",
) -> tuple:
    """Brings caches down to ``keep`` entries per KV head by their accumulated weights.

    A cache longer than ``keep`` keeps its first ``sinks`` and last ``recent`` entries and the
    ``keep - sinks - recent`` heaviest of the others (equal weights: the lower slot; NaN
    counts as the smallest), in their order; a shorter one is copied.

    Args:
        key/value: 16-bit ``[B, Hk, C, D]`` ("bhsd") or ``[B, C, Hk, D]`` ("bshd").
        weights: fp32 ``[B, Hk, C]`` with unit slot stride.
        lengths: int32 ``[B]`` entries of each cache.
        out: optional (key, value, weights) to write to, with at least ``keep`` slots and no
            memory of the inputs (two sets of caches can take turns); slots past ``keep`` stay
            as they are.  Default: new tensors of ``keep`` slots.

    Returns:
        (key, value, weights, lengths, index): the caches, ``min(lengths, keep)``, and the
        int32 ``[B, Hk, keep]`` slots the entries came from.  Slots from the new length up to
        ``keep`` are zero, with index -1.
    """
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"unsupported layout: {layout}")
    if not isinstance(key, torch.Tensor) or key.dim() != 4:
        raise ValueError("key cache must be a rank-4 tensor")
    if key.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"key cache must be fp16 or bf16, got {key.dtype}")
    B, D = key.shape[0], key.shape[3]
    Hk = key.shape[1] if layout == "bhsd" else key.shape[2]
    if weights is None:
        raise ValueError("weights are required")
    C = check_cache(key, value, lengths, weights, layout, B, Hk, D, key)
    if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"sinks ({sinks}) and recent ({recent}) must fit in keep ({keep})")
    _no_grad("evict_by_weight", key, value, weights)
    if out is not None:
        key_out, value_out, weights_out = out
        slots = check_cache(key_out, value_out, lengths, weights_out, layout, B, Hk, D, key)
        if weights_out is None or slots < keep:
            raise ValueError(f"out must be (key, value, weights) with at least keep = {keep} slots")
        if key_out.stride(3) != 1 or value_out.stride(3) != 1:
            raise ValueError("out is written in place and needs unit head-dim stride")
        for x in out:
            if any(_overlap(x, y) for y in (key, value, weights, lengths)):
                raise ValueError("out may not share memory with the inputs")
    if not key.is_cuda:
        raise RuntimeError("evict_by_weight runs on CUDA (sm_100a) tensors only")
    device = key.device
    key = key if key.stride(3) == 1 else key.contiguous()
    value = value if value.stride(3) == 1 else value.contiguous()
    if out is None:
        shape = (B, Hk, keep, D) if layout == "bhsd" else (B, keep, Hk, D)
        key_out, value_out = torch.empty(shape, dtype=key.dtype, device=device), torch.empty(shape, dtype=key.dtype, device=device)
        weights_out = torch.empty((B, Hk, keep), dtype=torch.float32, device=device)
    lengths_out = torch.empty_like(lengths)
    index = torch.empty((B, Hk, keep), dtype=torch.int32, device=device)
    if B and Hk and D:
        args = _lib.EvictArgs(
            key.data_ptr(), value.data_ptr(), weights.data_ptr(), lengths.data_ptr(), key_out.data_ptr(),
            value_out.data_ptr(), weights_out.data_ptr(), lengths_out.data_ptr(), index.data_ptr(), _bth(key, layout),
            _bth(value, layout), weights.stride()[:2], _bth(key_out, layout), _bth(value_out, layout),
            weights_out.stride()[:2], B, C, Hk, D, keep, sinks, recent)
        _lib.launch("fa4d_evict", args, device)
    return key_out, value_out, weights_out, lengths_out, index


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether the memory spans of two tensors meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    if x.numel() == 0 or y.numel() == 0:
        return False
    (a, b), (c, d) = span(x), span(y)
    return a < d and c < b


__all__ = ["shared_prefix_attention", "evict_by_weight"]
