"""Decoding for a batch of requests behind one shared prompt, with caches of bounded size.

One attention layer with random weights: the shared prompt goes through the flash attention
once (rotary positions with three axes: text, then an image's patches); then every step each
request's new token is rotated and appended to its cache, attends over the shared prompt and
its own cache in one softmax while the weight each entry receives is added up, and caches that
run full are brought back to their budget.

    python examples/shared_prefix_decode.py [--batch 16] [--steps 64] [--check]

``--check`` compares every step with the same computation in plain torch (float32).
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from tilelang_fa2_4d_mask import (  # noqa: E402
    MultiAxisRotary,
    evict_by_weight,
    shared_prefix_attention,
    tilelang_flash_attention,
)


def prompt_positions(text: int, height: int, width: int) -> torch.Tensor:
    """[3, 1, T]: `text` tokens that count alike on all axes, then the patches of an image."""
    n = height * width
    i = torch.arange(n)
    image = torch.stack([torch.zeros(n, dtype=torch.long), i // width, i % width]) + text
    return torch.cat([torch.arange(text).expand(3, -1), image], 1)[:, None]


class Layer:
    """An attention layer's projections, random."""

    def __init__(self, dim, heads, kv_heads, head_dim, dtype, device, generator):
        def w(rows, cols):
            return (torch.randn(rows, cols, generator=generator) * rows ** -0.5).to(device, dtype)

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.wq, self.wk, self.wv = w(dim, heads * head_dim), w(dim, kv_heads * head_dim), w(dim, kv_heads * head_dim)
        self.wo = w(heads * head_dim, dim)
        self.rotary = MultiAxisRotary(head_dim, (head_dim // 8, head_dim // 2 - head_dim // 8 - head_dim // 4, head_dim // 4))

    def qkv(self, x):
        """x [B, T, dim] -> q [B, T, Hq, D], k and v [B, T, Hk, D]."""
        B, T, _ = x.shape
        return ((x @ self.wq).view(B, T, self.heads, -1), (x @ self.wk).view(B, T, self.kv_heads, -1),
                (x @ self.wv).view(B, T, self.kv_heads, -1))


@torch.no_grad()
def decode(batch=16, steps=64, capacity=96, keep=64, sinks=2, recent=24, text=200, image=(12, 16), heads=8, kv_heads=2,
           head_dim=128, dim=256, dtype=torch.bfloat16, device="cuda", seed=0, observe=None):
    """Runs the loop; returns the last hidden states [batch, dim], the new caches' lengths and
    the seconds of the steps.  `observe(step, layer, prefix, q, cache, out)` sees every step."""
    g = torch.Generator().manual_seed(seed)
    layer = Layer(dim, heads, kv_heads, head_dim, dtype, device, g)

    # The shared prompt, once.
    positions = prompt_positions(text, *image).to(device)
    prompt = torch.randn(1, positions.shape[2], dim, generator=g).to(device, dtype)
    q, k, v = layer.qkv(prompt)
    q, k = layer.rotary(q, k, positions, layout="bshd")
    out = tilelang_flash_attention(q, k, v, is_causal=True, layout="bshd")
    prefix_key, prefix_value = k[0], v[0]  # [P, Hk, D]
    x = (out[0, -1].reshape(1, -1) @ layer.wo + torch.randn(batch, dim, generator=g).to(device, dtype))

    # Two sets of caches that take turns: eviction copies from one to the other.
    def new_cache():
        return [torch.zeros(batch, capacity, kv_heads, head_dim, dtype=dtype, device=device) for _ in range(2)] + [
            torch.zeros(batch, kv_heads, capacity, device=device)]

    cache, spare = new_cache(), new_cache()
    lengths = torch.zeros(batch, dtype=torch.int32, device=device)
    used = 0  # the longest cache, known without asking the device
    at = int(positions.max()) + 1
    torch.cuda.synchronize()
    began = time.perf_counter()
    for step in range(steps):
        if used == capacity:
            *spare[:], lengths, _ = evict_by_weight(*cache, lengths, keep=keep, sinks=sinks, recent=recent, out=tuple(spare),
                                                    layout="bshd")
            cache, spare, used = spare, cache, keep
        q, k, v = layer.qkv(x[:, None])
        now = torch.full((3, 1, 1), at + step, dtype=torch.long, device=device)
        q, lengths = layer.rotary.append(q, k, v, now, cache[0], cache[1], lengths, weights=cache[2], layout="bshd")
        used += 1
        before = cache[2].clone() if observe else None
        out = shared_prefix_attention(q, prefix_key, prefix_value, cache[0], cache[1], lengths, weights=cache[2], layout="bshd")
        if observe:
            observe(step, (prefix_key, prefix_value), q, (*cache, lengths, before), out)
        x = torch.tanh(out.reshape(batch, -1) @ layer.wo)
    torch.cuda.synchronize()
    return x, lengths, time.perf_counter() - began


def compare(step, prefix, q, cache, out):
    """The step's attention in plain torch, float32: asserts that output and weights agree."""
    key, value, weights, lengths, before = cache
    B, _, Hq, D = q.shape
    P, Hk = prefix[0].shape[:2]
    q = q[:, 0].float().view(B, Hk, Hq // Hk, D) * D ** -0.5
    logits = torch.cat([torch.einsum("bhgd,phd->bhgp", q, prefix[0].float()),
                        torch.einsum("bhgd,bjhd->bhgj", q, key.float())], -1)
    late = torch.arange(key.shape[1], device=key.device) >= lengths[:, None]
    logits[..., P:].masked_fill_(late[:, None, None], float("-inf"))
    p = logits.softmax(-1)
    want = torch.einsum("bhgp,phd->bhgd", p[..., :P], prefix[1].float()) + torch.einsum("bhgj,bjhd->bhgd", p[..., P:], value.float())
    error = (out.float().view_as(want) - want).abs().max()
    gained = (weights - before - p[..., P:].sum(2)).abs().max()
    # bf16 probabilities and output, values of order one; weights in 32 bits.
    assert float(error) < 0.04 and float(gained) < 1e-4, (step, float(error), float(gained))


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    decode(a.batch, 4)  # warm-up
    x, lengths, seconds = decode(a.batch, a.steps, observe=compare if a.check else None)
    print(f"{a.steps} steps of {a.batch} requests: {seconds / a.steps * 1e6:.0f} us a step, "
          f"caches of {int(lengths.min())} entries{', every step agrees with plain torch' if a.check else ''}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
