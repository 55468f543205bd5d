"""Serving: attention of a batch's new tokens over a prefix that all requests share and each
request's own cache, and eviction from the caches by the attention weight their entries
received.

A decode step rotates and appends the new tokens (``MultiAxisRotary.append``), attends
(``shared_prefix_attention``, which can accumulate ``weights``) and, when caches run full,
shrinks them (``evict_by_weight``).  Everything is enqueued on the current stream without a
host synchronisation, so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .rotary import Layout


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
            received, summed over the group's query heads and the T tokens.  The workspace then
            holds the own keys' logits, ``4 * B * Hq * T * C`` bytes by the caches' capacity C.
        scale: softmax scale, ``head_dim ** -0.5`` by default.
        is_causal: new token t sees the own entries up to its own, ``lengths - T + t``.

    Returns:
        The output in the query's layout; rows that see no key are 0.  A row that sees a NaN, or
        whose every logit is -inf, is NaN, as its softmax is; what no token of the request may see
        can hold anything.

    Rows that are not on 16-byte boundaries are copied first.  There is no gradient, in either
    mode; ``weights`` is written as by an in-place operation.
    """
    return _lib.host().shared_prefix_attention(query, prefix_key, prefix_value, key, value, lengths, mask, weights, scale,
                                               is_causal, layout)


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
            element of the inputs or of each other (two sets of caches can take turns); slots
            past ``keep`` stay as they are.  Default: new tensors of ``keep`` slots.

    Returns:
        (key, value, weights, lengths, index): the caches, ``min(lengths, keep)``, and the
        int32 ``[B, Hk, keep]`` slots the entries came from.  Slots from the new length up to
        ``keep`` are zero, with index -1.
    """
    return _lib.host().evict_by_weight(key, value, weights, lengths, keep, sinks, recent, out, layout)


__all__ = ["shared_prefix_attention", "evict_by_weight"]
