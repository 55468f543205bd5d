"""Plain restatements of norms before the rotary turn and of caches in 8 bits, in 64 bits."""

from __future__ import annotations

import math

import torch

from .serving import rotary_ref

BLOCK = 64
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def norm_ref(x, weight, eps):
    """Heads x [..., D] normalised, differentiable."""
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def norm_rotary_grads(x, weight, dy, positions, sections, *, eps, **kw):
    """(turn^-1(dy), dx, dw) of the norm and turn, by the formula."""
    x, w = x.double(), weight.double()
    g = rotary_ref(dy, positions, sections, inverse=True, **kw)
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    dx = r * (w * g - x * r ** 2 * (w * g * x).mean(-1, keepdim=True))
    return g, dx, (g * x * r).sum((0, 1, 2))


def least_scale(most, dtype):
    """The least 2^e, e >= -126, with most <= largest code * 2^e; NaN where most is not finite."""
    if not math.isfinite(most):
        return math.nan
    e = -126
    while most > LARGEST[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest_code(x, dtype):
    """x (64 bits, within the largest code) at the nearest value of a code, ties to even."""
    if dtype == torch.int8:
        return torch.round(x)
    e = torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent.long() - 1
    step = (e - 3 + 1023 << 52).view(torch.float64)  # 2^(e - 3), by its bits: powers on a GPU are not exact
    return torch.round(x / step) * step


def join_block(codes, scale, fresh, had, dtype):
    """A block [<= 64, D] of which `had` entries are held, and the fresh values that join behind
    them: (codes as values, scale)."""
    new = least_scale(float(fresh.abs().max()) if torch.isfinite(fresh).all() else math.inf, dtype)
    if had:
        new = math.nan if math.isnan(new) or math.isnan(scale) else max(new, scale)
    held = codes[:had].double()
    if had and new > scale:
        held = nearest_code(held * (scale / new), dtype)
    joined = torch.zeros_like(fresh) if math.isnan(new) else nearest_code(fresh / new, dtype)
    return torch.cat([held, joined]), new


def values_ref(codes, scale, lengths):
    """Canonical codes [B, Hk, C, D], scale [B, Hk, blocks] -> values in 64 bits, 0 past the lengths."""
    C = codes.shape[2]
    v = codes.to(torch.float64) * scale.double().repeat_interleave(BLOCK, 2)[:, :, :C, None]
    past = torch.arange(C, device=codes.device) >= lengths.long()[:, None]
    return v.masked_fill(past[:, None, :, None], 0.0)
