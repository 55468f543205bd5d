"""Rotary positions with several axes, for queries and keys on their way to the attention.

``MultiAxisRotary`` turns pairs of a head's elements by angles that grow with the token's
position; each pair follows one of several position axes (time, height and width of a
video's patches, say), ``sections`` giving the number of pairs of each axis in order.  Text
has the same position on every axis.  Each head can be normalised first, in the same pass.
Calling it is differentiable; ``append`` is the serving form, which also stores the turned keys
and the values in a cache of 16 or 8 bits.
"""

from __future__ import annotations

import math
from typing import Literal, Optional, Sequence

import torch

from . import _lib

Layout = Literal["bhsd", "bshd"]
_PAIRINGS = {"half": _lib.PAIR_HALF, "adjacent": _lib.PAIR_ADJACENT}


class MultiAxisRotary:
    """Rotary positions with one or more axes.

    Args:
        head_dim: size of a head, even, at most 256.
        sections: pairs of each axis, in order; they add up to ``rotary_dim / 2``.
        base: pair i turns by ``base ** (-2 i / rotary_dim)`` radians per position.
        rotary_dim: elements of a head that are turned (default all); the rest is copied.
        pairing: "half" pairs element i with i + rotary_dim / 2, "adjacent" 2 i with 2 i + 1.

    Positions are integers and may be negative.  The product of position and frequency is exact
    modulo a turn, so an angle is off by at most 2**-25 turns, and ``1.2 * abs(position) * 2**-64``
    for the rounding of the frequency (for a base of 1 or more).  Objects can be copied and pickled.
    """

    # Where a process that loads a pickle finds it: this package has no importable name of its own.
    __module__ = "tilelang_fa2_4d_mask"

    def __init__(self, head_dim: int, sections: Sequence[int], *, base: float = 10000.0,
                 rotary_dim: Optional[int] = None, pairing: str = "half"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim % 2 or head_dim > 2 * _lib.ROTARY_MAX_PAIRS:
            raise ValueError(f"head_dim must be even and at most {2 * _lib.ROTARY_MAX_PAIRS}, got {head_dim}")
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be even and at most head_dim, got {rotary_dim}")
        sections = tuple(int(n) for n in sections)
        if not sections or len(sections) > 255 or min(sections) < 0 or sum(sections) != rotary_dim // 2:
            raise ValueError(f"sections must add up to rotary_dim / 2 = {rotary_dim // 2}, got {sections}")
        if pairing not in _PAIRINGS:
            raise ValueError(f"unsupported pairing: {pairing}")
        if not (math.isfinite(base) and base > 0):
            raise ValueError(f"base must be positive, got {base}")
        self.head_dim, self.sections, self.base = head_dim, sections, float(base)
        self.rotary_dim, self.pairing = rotary_dim, pairing
        self._make_table()

    def _make_table(self) -> None:
        self._host = _lib.host()
        self._table = self._host.make_table(self.base, self.sections, self.head_dim, self.rotary_dim, _PAIRINGS[self.pairing])

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k not in ("_host", "_table")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._make_table()

    def __call__(self, query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, *,
                 query_norm: Optional[torch.Tensor] = None, key_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 layout: Layout = "bhsd") -> tuple:
        """Turned (query, key), differentiable in both, and in the norms' weights.

        Args:
            query/key: fp16/bf16 ``[B, H, T, D]`` ("bhsd") or ``[B, T, H, D]`` ("bshd"), any
                strides; their head counts may differ.
            positions: integer ``[axes, B or 1, T]`` (int32 and int64 are read as they are).
            query_norm/key_norm: weights ``[D]``, both fp32 or both in the tokens' dtype: each head x
                becomes ``x * (mean(x**2) + eps) ** -0.5 * weight`` (in 32 bits, squares included)
                before it is turned.  Gradients have no gradients of their own then.  Cosines and
                sines are off by at most 2**-23 in this form.
        """
        if query_norm is None and key_norm is None:
            return self._host.rotary(self._table, query, key, positions, layout)
        return self._host.norm_rotary(self._table, query, key, positions, query_norm, key_norm, eps, layout)

    def append(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
               key_cache: torch.Tensor, value_cache: torch.Tensor, lengths: torch.Tensor, *,
               weights: Optional[torch.Tensor] = None, query_norm: Optional[torch.Tensor] = None,
               key_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, key_scale: Optional[torch.Tensor] = None,
               value_scale: Optional[torch.Tensor] = None, layout: Layout = "bhsd") -> tuple:
        """Turns the new tokens' query and key (normalised first, as in a call, where ``query_norm``
        and ``key_norm`` are given) and stores key and value in the caches.

        Args:
            query/key/value: the T new tokens, as for a call (value has the key's heads).
            positions: integer ``[axes, B or 1, T]``.
            key_cache/value_cache: ``[B, Hk, C, D]`` ("bhsd") or ``[B, C, Hk, D]`` ("bshd"),
                written in place at slots ``lengths[b] .. lengths[b] + T - 1``.
            lengths: int32 ``[B]`` entries of each cache so far.
            weights: optional fp32 ``[B, Hk, C]`` attention weights of the cache entries, set
                to 0 at the new slots.
            key_scale/value_scale: of caches held in 8 bits (``torch.float8_e4m3fn`` or ``torch.int8``
                codes, head dim a multiple of 16, rows on 16-byte boundaries, no ``weights``): fp32
                ``[B, Hk, ceil(C / 64)]``, a scale for each 64 slots of a request and head,
                updated in place.  A value is its code times its block's scale.  Scales written here
                are powers of two: the least, 2**-126 or more, under which no value of the block
                passes the largest code (448 or 127).  Where new tokens raise a block's scale, its
                earlier codes are rounded anew; it does not sink until its first slot is written
                again.  An infinity or NaN makes its block's scale NaN, and so the whole block.
                The caches and scales may not share memory.  Cosines and sines are those of the form
                with norms, with or without them: the query can differ in its last bit from a call's.

        Returns:
            (turned query, new lengths).  Tokens past the capacity C are not stored: the new
            length stays at C and ``DEV_CACHE_FULL`` is set in ``device_status()``.
        """
        if query_norm is None and key_norm is None and key_scale is None and value_scale is None:
            return self._host.rotary_append(self._table, query, key, value, positions, key_cache, value_cache, lengths,
                                            weights, layout)
        return self._host.norm_append(self._table, query, key, value, positions, key_cache, value_cache, lengths, weights,
                                      query_norm, key_norm, eps, key_scale, value_scale, layout)


__all__ = ["MultiAxisRotary"]
