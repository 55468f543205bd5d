"""Plain 64-bit restatements of the operators around the attention: rotary positions with
several axes, attention over a shared prefix and own caches, eviction by weight."""

from __future__ import annotations

import math

import torch


def rotary_ref(x, positions, sections, *, base, rotary_dim=None, pairing="half", inverse=False, layout="bhsd"):
    """x [B, H, T, D] or [B, T, H, D] turned by positions [axes, B or 1, T], in float64."""
    x = x.double()
    if layout == "bhsd":
        x = x.transpose(1, 2)
    D = x.shape[-1]
    R = D if rotary_dim is None else rotary_dim
    y = x.clone()
    pair = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            phi = positions[axis].double() * base ** (-2.0 * pair / R)
            phi = phi.expand(x.shape[0], -1).unsqueeze(-1)
            c, s = torch.cos(phi), torch.sin(phi) * (-1.0 if inverse else 1.0)
            i, j = (pair, pair + R // 2) if pairing == "half" else (2 * pair, 2 * pair + 1)
            y[..., i] = x[..., i] * c - x[..., j] * s
            y[..., j] = x[..., j] * c + x[..., i] * s
            pair += 1
    return y.transpose(1, 2) if layout == "bhsd" else y


def shared_prefix_ref(q, pk, pv, k, v, lengths, *, mask=None, scale=None, causal=True):
    """Canonical layouts q [B, Hq, T, D], pk/pv [Hk, P, D] or None, k/v [B, Hk, C, D]; returns
    (out [B, Hq, T, D], probabilities of the own keys summed over group and tokens
    [B, Hk, C], sum of p |v| [B, Hq, T, D], the largest sum of |q k| * |scale| of the own and
    prefix logits), in float64.  Entries that no row may see are not read."""
    B, Hq, T, D = q.shape
    Hk, C = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    weights = torch.zeros(B, Hk, C, dtype=torch.float64, device=q.device)
    biggest = 0.0
    for b in range(B):
        n = min(max(int(lengths[b]), 0), C)
        for h in range(Hq):
            hk = h // G
            for t in range(T):
                lim = n - T + t + 1 if causal else n
                seen = torch.arange(C, device=q.device) < lim
                if mask is not None:
                    seen &= mask[b % mask.shape[0], h % mask.shape[1], t]
                idx = seen.nonzero().flatten()
                keys, vals = k[b, hk, idx].double(), v[b, hk, idx].double()
                if pk is not None:
                    keys, vals = torch.cat([pk[hk].double(), keys]), torch.cat([pv[hk].double(), vals])
                if len(keys) == 0:
                    continue
                row = q[b, h, t].double()
                p = torch.softmax(keys @ row * scale, 0)
                biggest = max(biggest, float((keys.abs() @ row.abs()).max()) * abs(scale))
                out[b, h, t] = p @ vals
                size[b, h, t] = p @ vals.abs()
                if len(idx):
                    weights[b, hk, idx] += p[len(p) - len(idx):]
    return out, weights, size, biggest


def evict_ref(weights, lengths, keep, sinks, recent):
    """Kept slots per (b, hk): int64 [B, Hk, keep], -1 past the new length."""
    w = weights.double().cpu()
    B, Hk, C = w.shape
    index = torch.full((B, Hk, keep), -1, dtype=torch.int64)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), C)
        for h in range(Hk):
            if n <= keep:
                chosen = list(range(n))
            else:
                rank = lambda j: -math.inf if math.isnan(w[b, h, j]) else float(w[b, h, j])  # noqa: E731
                nan = lambda j: math.isnan(w[b, h, j])  # noqa: E731
                middle = sorted(range(sinks, n - recent), key=lambda j: (-rank(j), nan(j), j))
                chosen = sorted([*range(sinks), *middle[: keep - sinks - recent], *range(n - recent, n)])
            index[b, h, : len(chosen)] = torch.tensor(chosen, dtype=torch.int64)
    return index
