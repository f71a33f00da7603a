"""PagedFp8KVCache: pages taken, moved and freed, and the decode example that uses every operator."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from helpers import np_bytes, np_values
from oracle import paged_kv as opk

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def pk():
    from kernel_agent_b200.kernels import paged_kv

    return paged_kv


def attention_of(cache, q):
    want, _, size = opk.attention(np_values(q), np_bytes(cache.k_pages), np_values(cache.k_scale), np_bytes(cache.v_pages),
                                  np_values(cache.v_scale), cache.page_table.cpu().numpy(), cache.tokens)
    return want, size


def test_life_of_a_cache(pk):
    """Prompts of unequal length, tokens, evictions and a freed sequence: the pages stay apart, the
    lengths agree, and the attention is that of what the pages hold."""
    cache = pk.PagedFp8KVCache(3, 2, 64, num_pages=40, page_tokens=16)
    g = torch.Generator(device=DEV).manual_seed(0)
    draw = lambda t: torch.randn(3, 2, t, 64, generator=g, device=DEV)  # noqa: E731
    cache.append(draw(70), draw(70), counts=[70, 0, 33])
    for step in range(40):
        cache.append(draw(1), draw(1), counts=None if step % 3 else [1, 1, 0])
        q = torch.randn(3, 4, 1, 64, generator=g, device=DEV)
        out = cache.attend(q)
        if step % 8 == 0:
            want, size = attention_of(cache, q)
            # fp32 queries: 22 bits of the weights and a score's fp32 roundings
            assert np.all(np.abs(np_values(out) - want) <= 2.0 ** -14 * size)
        if step == 20:
            over, kept = cache.evict(50, recent=10, sinks=2)
            assert over == [0] and cache.tokens[0] == 50 and kept.shape == (1, 2, 50)
            assert kept[0, :, :2].tolist() == [[0, 1]] * 2 and kept[0, 0, -1].item() == 90
            assert cache.evict(500) == ([], None)
        if step == 30:
            cache.free(2)
            assert cache.tokens[2] == 0
        assert cache.lengths.tolist() == cache.tokens
        held = [p for pages in cache._pages for p in pages]
        assert len(held) == len(set(held)) and sorted(held + cache._free) == list(range(40))
        assert [len(p) for p in cache._pages] == [-(-n // 16) for n in cache.tokens]


def test_reserve_and_capture(pk):
    """A captured step appends and attends through the pool's tensors after a reserve."""
    cache = pk.PagedFp8KVCache(2, 2, 128, num_pages=12, page_tokens=32)
    x = torch.randn(2, 2, 30, 128, device=DEV).to(torch.bfloat16)
    cache.append(x, x)
    cache.reserve([40, 40])
    q = torch.randn(2, 2, 1, 128, device=DEV).to(torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="reserve"):
            cache.append(x[:, :, :1], x[:, :, :1])
        pk.append_kv_pages(x[:, :, :1], x[:, :, :1], *cache.pool, mass=cache.mass, out_lengths=cache.lengths)
        out = pk.paged_kv_attention(q, *cache.pool, mass=cache.mass)
    for i in range(40):
        graph.replay()
    assert cache.lengths.tolist() == [70, 70]
    assert torch.equal(out, pk.paged_kv_attention(q, *cache.pool))


def test_refusals(pk):
    for args, match in (((1, 1, 96, 4), "head_dim"), ((1, 1, 64, 4, 24), "page_tokens")):
        with pytest.raises(ValueError, match=match):
            pk.PagedFp8KVCache(*args)
    with pytest.raises(ValueError, match="CUDA"):
        pk.PagedFp8KVCache(1, 1, 64, 4, device="cpu")
    cache = pk.PagedFp8KVCache(2, 1, 64, num_pages=4, page_tokens=16, max_pages=3, mass=False)
    x = torch.zeros(2, 1, 64, 64, device=DEV)
    with pytest.raises(ValueError, match="full"):
        cache.append(x, x)
    with pytest.raises(ValueError, match="pass 3 pages"):
        cache.append(x, x, counts=[49, 0])
    with pytest.raises(ValueError, match="counts"):
        cache.append(x, x, counts=[65, 0])
    with pytest.raises(ValueError, match="counts"):
        cache.reserve([1])
    with pytest.raises(ValueError, match="mass"):
        cache.evict(8)
    assert cache.tokens == [0, 0] and cache.free_pages == 4
    cache = pk.PagedFp8KVCache(1, 1, 64, num_pages=4, page_tokens=16)
    cache.append(x[:1], x[:1])
    with pytest.raises(ValueError, match="full"):
        cache.evict(20)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(8, recent=9)


def test_decode_example():
    """The example runs every operator; FP4 weights and an FP8 cache stay near bf16 (NVFP4's rounding is
    about 0.1 of a weight), and the cache keeps to its budget."""
    path = Path(__file__).resolve().parents[1] / "examples" / "decode_fp4.py"
    spec = importlib.util.spec_from_file_location("decode_fp4", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    before, after, cache = example.decode(example.Layer(hidden=256, heads=4, kv_heads=2, head_dim=64, inner=512), 60, 48, 3)
    assert 0.0 < before < 0.25 and before > 0.01 and after < 0.5
    assert max(cache.tokens) <= 60 and cache.lengths.tolist() == cache.tokens
