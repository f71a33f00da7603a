"""Decoding with FP4 weights and a paged FP8 cache of a fixed budget: one decoder layer, token by token.

    python examples/decode_fp4.py [--tokens 256] [--budget 192] [--batch 2]

The layer's weights are quantised once with ``quantize_fp4``; the prompt and every token go through
``fp4_w4a16_linear``, their keys and values into a ``PagedFp8KVCache``, and whenever a sequence passes
the budget by a quarter it is cut back to it by the weights its tokens received. The same tokens go
through the layer with its bf16 weights and a full bf16 cache; the difference is printed.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "kernel-agent_b200"))

from kernel_agent_b200.kernels.gemv import fp4_w4a16_linear  # noqa: E402
from kernel_agent_b200.kernels.paged_kv import PagedFp8KVCache  # noqa: E402
from kernel_agent_b200.kernels.quant import quantize_fp4  # noqa: E402


class Layer:
    """Attention and a gated MLP with residuals; weights in bf16 and in NVFP4."""

    def __init__(self, hidden=1024, heads=8, kv_heads=2, head_dim=128, inner=2048, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        sizes = {"q": (heads * head_dim, hidden), "k": (kv_heads * head_dim, hidden), "v": (kv_heads * head_dim, hidden),
                 "o": (hidden, heads * head_dim), "gate": (inner, hidden), "up": (inner, hidden), "down": (hidden, inner)}
        self.weights = {name: (torch.randn(size, generator=g, device=device) * size[1] ** -0.5).to(torch.bfloat16)
                        for name, size in sizes.items()}
        self.fp4 = {name: quantize_fp4(w) for name, w in self.weights.items()}

    def linear(self, name, x, fp4):
        if fp4:
            return fp4_w4a16_linear(x, *self.fp4[name])
        return torch.nn.functional.linear(x, self.weights[name])

    def split(self, x, heads):  # [batch, tokens, heads * dim] -> [batch, heads, tokens, dim]
        return x.unflatten(-1, (heads, self.head_dim)).transpose(1, 2)

    def forward(self, x, attention, fp4):
        """``x [batch, tokens, hidden]``; ``attention(q, k, v)`` keeps the cache."""
        h = torch.nn.functional.rms_norm(x, x.shape[-1:])
        q = self.split(self.linear("q", h, fp4), self.heads)
        k, v = self.split(self.linear("k", h, fp4), self.kv_heads), self.split(self.linear("v", h, fp4), self.kv_heads)
        x = x + self.linear("o", attention(q, k, v).transpose(1, 2).flatten(2), fp4)
        h = torch.nn.functional.rms_norm(x, x.shape[-1:])
        gate = torch.nn.functional.silu(self.linear("gate", h, fp4))
        return x + self.linear("down", gate * self.linear("up", h, fp4), fp4)


def decode(layer: Layer, tokens: int, budget: int, batch: int, prompt: int = 32, page_tokens: int = 32, seed: int = 1):
    """Runs a prompt and ``tokens`` single tokens both ways; returns the largest relative difference of
    a step's output while nothing had been evicted, the same afterwards, and the cache."""
    device = layer.weights["q"].device
    g = torch.Generator(device=device).manual_seed(seed)
    hidden = layer.weights["q"].shape[1]
    # tokens drawn from a small vocabulary, so that earlier ones matter to later ones
    vocabulary = torch.randn(64, hidden, generator=g, device=device).to(torch.bfloat16)
    ids = torch.randint(0, 64, (batch, prompt + tokens), generator=g, device=device)
    room = -(-(budget + budget // 4 + 1) // page_tokens) + -(-budget // page_tokens)
    cache = PagedFp8KVCache(batch, layer.kv_heads, layer.head_dim, batch * room + 2, page_tokens, device=device)
    full = []

    def paged(q, k, v):
        cache.append(k, v)
        return cache.attend(q)

    def plain(q, k, v):
        if full:
            k, v = torch.cat([full[0], k], 2), torch.cat([full[1], v], 2)
        full[:] = [k, v]
        seen = torch.ones(q.shape[2], k.shape[2], dtype=torch.bool, device=device).tril(k.shape[2] - q.shape[2])
        return torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=seen, enable_gqa=True)

    worst = [0.0, 0.0]
    evicted = False
    at = 0
    for size in [prompt] + [1] * tokens:
        x = vocabulary[ids[:, at:at + size]]
        at += size
        got = layer.forward(x, paged, True)
        want = layer.forward(x, plain, False)
        difference = float((got.float() - want.float()).norm() / want.float().norm())
        worst[evicted] = max(worst[evicted], difference)
        if max(cache.tokens) > budget + budget // 4:
            cache.evict(budget, recent=budget // 4, sinks=4)
            evicted = True
    return worst[0], worst[1], cache


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=256)
    parser.add_argument("--budget", type=int, default=192)
    parser.add_argument("--batch", type=int, default=2)
    a = parser.parse_args()
    before, after, cache = decode(Layer(), a.tokens, a.budget, a.batch)
    print(f"{a.tokens} tokens x {a.batch} sequences; cached now: {cache.tokens}; free pages: {cache.free_pages}")
    print(f"relative difference to bf16 weights and a full bf16 cache: {before:.3f} before the first eviction, "
          f"{after:.3f} after it")


if __name__ == "__main__":
    main()
