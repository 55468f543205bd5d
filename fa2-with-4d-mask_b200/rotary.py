"""Rotary positions with several axes, for queries and keys on their way to the attention.

``MultiAxisRotary`` turns pairs of a head's elements by angles that grow with the token's
position; each pair follows one of several position axes (time, height and width of a
video's patches, say), ``sections`` giving the number of pairs of each axis in order.  Text
has the same position on every axis.  Calling it is differentiable; ``append`` is the
serving form, which also stores the turned keys and the values in a cache.
"""

from __future__ import annotations

import math
from typing import Literal, Optional, Sequence

import torch

from . import _lib

Layout = Literal["bhsd", "bshd"]
_PAIRINGS = {"half": _lib.PAIR_HALF, "adjacent": _lib.PAIR_ADJACENT}


def _bth(x: torch.Tensor, layout: str) -> tuple:
    """(batch, seq, head) strides of a rank-4 tensor in the given layout."""
    s = x.stride()
    return (s[0], s[2], s[1]) if layout == "bhsd" else s[:3]


def _check_tokens(tensors, layout: str, head_dim: int) -> tuple:
    """Validates [B, H, T, D] / [B, T, H, D] tensors of one dtype, device, B, T and head dim:
    (query, key) or (query, key, value), value with the key's heads; returns (B, T, Hq, Hk)."""
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"unsupported layout: {layout}")
    seq = 2 if layout == "bhsd" else 1
    query, key = tensors[:2]
    for name, x in zip(("query", "key", "value"), tensors):
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError(f"{name} must be a rank-4 tensor")
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"{name} must be fp16 or bf16, got {x.dtype}")
        if x.dtype != query.dtype or x.device != query.device:
            raise ValueError(f"{name} must have the dtype and device of query")
        if x.shape[0] != query.shape[0] or x.shape[seq] != query.shape[seq]:
            raise ValueError(f"{name} must have the batch size and sequence length of query")
        if x.shape[3] != head_dim:
            raise ValueError(f"{name} has head dimension {x.shape[3]}, expected {head_dim}")
    if tensors[-1].shape != key.shape:
        raise ValueError("value must have the heads of key")
    return query.shape[0], query.shape[seq], query.shape[3 - seq], key.shape[3 - seq]


def _need_cuda(x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError("MultiAxisRotary runs on CUDA (sm_100a) tensors only")


def _unit_rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(3) == 1 else x.contiguous()


class MultiAxisRotary:
    """Rotary positions with one or more axes.

    Args:
        head_dim: size of a head, even, at most 256.
        sections: pairs of each axis, in order; they add up to ``rotary_dim / 2``.
        base: pair i turns by ``base ** (-2 i / rotary_dim)`` radians per position.
        rotary_dim: elements of a head that are turned (default all); the rest is copied.
        pairing: "half" pairs element i with i + rotary_dim / 2, "adjacent" 2 i with 2 i + 1.

    Angles are exact for every position (fixed point modulo a turn); positions are integers
    and may be negative.
    """

    def __init__(self, head_dim: int, sections: Sequence[int], *, base: float = 10000.0,
                 rotary_dim: Optional[int] = None, pairing: str = "half"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim % 2 or head_dim > 2 * _lib.ROTARY_MAX_PAIRS:
            raise ValueError(f"head_dim must be even and at most {2 * _lib.ROTARY_MAX_PAIRS}, got {head_dim}")
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be even and at most head_dim, got {rotary_dim}")
        sections = tuple(int(n) for n in sections)
        if not sections or min(sections) < 0 or sum(sections) != rotary_dim // 2:
            raise ValueError(f"sections must add up to rotary_dim / 2 = {rotary_dim // 2}, got {sections}")
        if pairing not in _PAIRINGS:
            raise ValueError(f"unsupported pairing: {pairing}")
        if not (math.isfinite(base) and base > 0):
            raise ValueError(f"base must be positive, got {base}")
        self.head_dim, self.sections, self.base = head_dim, sections, float(base)
        self.rotary_dim, self.pairing = rotary_dim, pairing
        t = self._table = _lib.RotaryTable()
        t.D, t.rotary_dim, t.pairing, t.axes = head_dim, rotary_dim, _PAIRINGS[pairing], len(sections)
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        for i in range(rotary_dim // 2):
            turns = self.base ** (-2.0 * i / rotary_dim) / (2.0 * math.pi)
            t.turn[i] = int(math.fmod(turns, 1.0) * 2.0 ** 64) & (2 ** 64 - 1)
            t.axis[i] = axis[i]

    def _positions(self, positions: torch.Tensor, B: int, T: int, device) -> tuple:
        """(tensor, strides (axis, batch, seq), bits) of [axes, B or 1, T] integer positions."""
        axes = len(self.sections)
        if not isinstance(positions, torch.Tensor) or positions.dim() != 3 or positions.shape[0] != axes \
                or positions.shape[1] not in (1, B) or positions.shape[2] != T:
            raise ValueError(f"positions must be an integer tensor of shape [{axes}, {B} or 1, {T}]")
        if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
            raise ValueError("positions must be an integer tensor")
        if positions.device != device:
            raise ValueError(f"positions must be on {device}, got {positions.device}")
        if positions.dtype not in (torch.int32, torch.int64):
            positions = positions.to(torch.int64)
        s = positions.stride()
        return positions, (s[0], 0 if positions.shape[1] == 1 else s[1], s[2]), 64 if positions.dtype == torch.int64 else 32

    def __call__(self, query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, *,
                 layout: Layout = "bhsd") -> tuple:
        """Turned (query, key), differentiable in both.

        Args:
            query/key: fp16/bf16 ``[B, H, T, D]`` ("bhsd") or ``[B, T, H, D]`` ("bshd"), any
                strides; their head counts may differ.
            positions: int32/int64 ``[axes, B or 1, T]``.
        """
        B, T, _, _ = _check_tokens((query, key), layout, self.head_dim)
        positions, strides, bits = self._positions(positions, B, T, query.device)
        _need_cuda(query)
        if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad):
            return _Rotate.apply(query, key, self, positions, strides, bits, layout)
        return self._rotate(query, key, positions, strides, bits, layout, 0)

    def _rotate(self, query, key, positions, strides, bits, layout, inverse) -> tuple:
        query, key = _unit_rows(query), _unit_rows(key)
        q_out, k_out = torch.empty_like(query), torch.empty_like(key)
        if query.shape[0] == 0 or query.shape[1] == 0 or query.shape[2] == 0 or key.numel() == 0:
            return q_out, k_out
        seq = 2 if layout == "bhsd" else 1
        args = _lib.RotaryArgs(
            self._table, query.data_ptr(), key.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), positions.data_ptr(),
            _bth(query, layout), _bth(key, layout), _bth(q_out, layout), _bth(k_out, layout), strides,
            query.shape[0], query.shape[seq], query.shape[3 - seq], key.shape[3 - seq], _lib._dtype_code(query.dtype),
            bits, inverse)
        _lib.launch("fa4d_rotary", args, query.device)
        return q_out, k_out

    def append(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
               key_cache: torch.Tensor, value_cache: torch.Tensor, lengths: torch.Tensor, *,
               weights: Optional[torch.Tensor] = None, layout: Layout = "bhsd") -> tuple:
        """Turns the new tokens' query and key and stores key and value in the caches.

        Args:
            query/key/value: the T new tokens, as for a call (value has the key's heads).
            positions: int32/int64 ``[axes, B or 1, T]``.
            key_cache/value_cache: ``[B, Hk, C, D]`` ("bhsd") or ``[B, C, Hk, D]`` ("bshd"),
                written in place at slots ``lengths[b] .. lengths[b] + T - 1``.
            lengths: int32 ``[B]`` entries of each cache so far.
            weights: optional fp32 ``[B, Hk, C]`` attention weights of the cache entries, set
                to 0 at the new slots.

        Returns:
            (turned query, new lengths).  Tokens past the capacity C are not stored: the new
            length stays at C and ``FA4D_DEV_CACHE_FULL`` is set in the device status word.
        """
        B, T, Hq, Hk = _check_tokens((query, key, value), layout, self.head_dim)
        positions, strides, bits = self._positions(positions, B, T, query.device)
        C = check_cache(key_cache, value_cache, lengths, weights, layout, B, Hk, self.head_dim, query)
        if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
            raise ValueError("append has no gradient: call it under torch.no_grad()")
        if key_cache.stride(3) != 1 or value_cache.stride(3) != 1:
            raise ValueError("the caches are written in place and need unit head-dim stride")
        _need_cuda(query)
        query, key, value = _unit_rows(query), _unit_rows(key), _unit_rows(value)
        q_out, lengths_out = torch.empty_like(query), torch.empty_like(lengths)
        if B == 0 or T == 0:
            return q_out, lengths.clone()
        args = _lib.RotaryAppendArgs(
            self._table, query.data_ptr(), key.data_ptr(), value.data_ptr(), q_out.data_ptr(), key_cache.data_ptr(),
            value_cache.data_ptr(), None if weights is None else weights.data_ptr(), positions.data_ptr(),
            lengths.data_ptr(), lengths_out.data_ptr(), _bth(query, layout), _bth(key, layout), _bth(value, layout),
            _bth(q_out, layout), _bth(key_cache, layout), _bth(value_cache, layout),
            (0, 0) if weights is None else weights.stride()[:2], strides, B, T, Hq, Hk, C,
            _lib._dtype_code(query.dtype), bits)
        _lib.launch("fa4d_rotary_append", args, query.device)
        return q_out, lengths_out


class _Rotate(torch.autograd.Function):
    """A turn by phi; its gradient is the turn by -phi."""

    @staticmethod
    def forward(ctx, query, key, rotary, positions, strides, bits, layout):
        ctx.save_for_backward(positions)
        ctx.rest = (rotary, strides, bits, layout)
        return rotary._rotate(query, key, positions, strides, bits, layout, 0)

    @staticmethod
    def backward(ctx, dq, dk):
        rotary, strides, bits, layout = ctx.rest
        return *rotary._rotate(dq, dk, *ctx.saved_tensors, strides, bits, layout, 1), None, None, None, None, None


def check_cache(key, value, lengths, weights, layout: str, B: int, Hk: int, head_dim: int, like: torch.Tensor) -> int:
    """Validates a batch's cache (key/value ``[B, Hk, C, D]`` or ``[B, C, Hk, D]``, lengths,
    optional weights) against B, Hk, head_dim and the dtype and device of `like`; returns C."""
    seq = 2 if layout == "bhsd" else 1
    for name, x in (("key cache", key), ("value cache", value)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError(f"{name} must be a rank-4 tensor")
        if x.dtype != like.dtype or x.device != like.device:
            raise ValueError(f"{name} must be {like.dtype} on {like.device}")
        if x.shape[0] != B or x.shape[3 - seq] != Hk or x.shape[3] != head_dim or x.shape[seq] != key.shape[seq]:
            raise ValueError(f"{name} has shape {tuple(x.shape)}, expected batch {B}, {Hk} heads of {head_dim} and "
                             "the same slots for keys and values")
    C = key.shape[seq]
    if C < 1:
        raise ValueError("the cache has no slots")
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,) \
            or lengths.device != like.device or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 tensor of shape [{B}] on {like.device}")
    if weights is not None:
        if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 \
                or tuple(weights.shape) != (B, Hk, C) or weights.device != like.device or weights.stride(2) != 1:
            raise ValueError(f"weights must be an fp32 tensor of shape {(B, Hk, C)} with unit slot stride on {like.device}")
    return C


__all__ = ["MultiAxisRotary"]
