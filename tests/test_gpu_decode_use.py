"""The decode operators as programs use them: from several threads, over shared pages, in captured
steps, on inputs of unusual layout."""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def pk():
    from kernel_agent_b200.kernels import paged_kv

    return paged_kv


@pytest.fixture(scope="module")
def gv():
    from kernel_agent_b200.kernels import gemv

    return gemv


def weight(n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8).to(DEV)
    return codes, torch.rand(n, k // 16, generator=g).add(0.5).to(E4M3).to(DEV)


def pool(pages, heads, page, dim, seed=0):
    """(k_pages, k_scale, v_pages, v_scale) of normal values."""
    g = torch.Generator().manual_seed(seed)
    codes = [(torch.randn(pages, heads, page, dim, generator=g) * 64).clamp(-448, 448).to(E4M3).to(DEV) for _ in range(2)]
    scale = torch.full((pages, heads), 2.0 ** -6, device=DEV)
    return codes[0], scale, codes[1], scale.clone()


def test_two_threads_on_one_stream(pk, gv):
    """Calls that two threads enqueue on the default stream give what each gives alone."""
    codes, scales = weight(4096, 4096)
    x = torch.randn(2, 8, 4096, device=DEV).to(torch.bfloat16)
    cache = pool(64, 2, 64, 128)
    table = torch.arange(64, dtype=torch.int32, device=DEV).reshape(1, 64)
    lengths = torch.tensor([4000], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 1, 8, 128, device=DEV).to(torch.bfloat16)
    ts = torch.tensor(0.01, device=DEV)

    def step(i):
        return gv.fp4_w4a16_linear(x[i], codes, scales, ts), pk.paged_kv_attention(q[i], *cache, table, lengths)

    want = [step(i) for i in range(2)]
    got = [[], []]

    def many(i):
        for _ in range(150):
            got[i].append(step(i))

    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 150
        for pair in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(pair, want[i]))


def test_append_past_the_reservation(pk):
    """Tokens past a sequence's pages are dropped and reported; no other sequence's page changes."""
    from kernel_agent_b200 import _native as nat

    cache = pk.PagedFp8KVCache(2, 1, 64, num_pages=6, page_tokens=16)
    x = torch.randn(2, 1, 16, 64, device=DEV)
    cache.append(x, x)
    before = [t.clone() for t in (cache.k_pages.view(torch.uint8), cache.k_scale, cache.mass)]
    pk.append_kv_pages(x * 8, x * 8, *cache.pool, mass=cache.mass)
    assert nat.device_status() == 2
    for a, b in zip(before, (cache.k_pages.view(torch.uint8), cache.k_scale, cache.mass)):
        assert torch.equal(a, b)
    assert nat.device_status() == 0


def test_captured_steps_then_others(pk):
    """Replays, their count, another reservation past it and plain appends: the host and the device agree,
    and what the other sequence holds stays."""
    cache = pk.PagedFp8KVCache(2, 1, 64, num_pages=16, page_tokens=16)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(2, 1, 20, 64, generator=g, device=DEV)
    cache.append(x, x)
    cache.reserve([30, 0])
    one = torch.randn(2, 1, 1, 64, generator=g, device=DEV)
    counts = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    held = cache._pages[1]
    before = cache.k_pages.view(torch.uint8)[held].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pk.append_kv_pages(one, one, *cache.pool, counts=counts, mass=cache.mass, out_lengths=cache.lengths)
    for _ in range(28):
        graph.replay()
    cache.advance([28, 0])
    assert cache.tokens == cache.lengths.tolist() == [48, 20]
    cache.reserve([20, 0])
    for _ in range(17):  # into the pages of the second reservation
        graph.replay()
    cache.advance([17, 0])
    cache.append(one, one, counts=[1, 0])
    assert cache.tokens == cache.lengths.tolist() == [66, 20]
    assert torch.equal(cache.k_pages.view(torch.uint8)[held], before)
    assert cache._pages[1] == held and len(set(cache._pages[0]) & set(held)) == 0
    over, _ = cache.evict(40)
    assert over == [0] and cache.tokens == cache.lengths.tolist() == [40, 20]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear_x_off_16_bytes(gv, dtype):
    codes, scales = weight(40, 128)
    for m in (1, 3):
        flat = torch.randn(1 + m * 128, device=DEV).to(dtype)
        x = flat[1:].view(m, 128)
        assert torch.equal(gv.fp4_w4a16_linear(x, codes, scales, 0.1), gv.fp4_w4a16_linear(x.clone(), codes, scales, 0.1))


def test_append_rows_off_16_bytes(pk):
    table = torch.arange(4, dtype=torch.int32, device=DEV).reshape(1, 4)
    lengths = torch.tensor([5], dtype=torch.int32, device=DEV)
    for new in (1, 20):
        flat = torch.randn(1 + new * 64, device=DEV).to(torch.bfloat16)
        off = flat[1:].view(1, 1, new, 64)
        got, want = pool(4, 1, 16, 64), pool(4, 1, 16, 64)
        pk.append_kv_pages(off, off, *got, table, lengths)
        pk.append_kv_pages(off.clone(), off.clone(), *want, table, lengths)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    odd = torch.randn(70, device=DEV).as_strided((1, 1, 1, 64), (70, 35, 70, 1))
    got, want = pool(4, 1, 16, 64), pool(4, 1, 16, 64)
    pk.append_kv_pages(odd, odd, *got, table, lengths)
    pk.append_kv_pages(odd.clone(memory_format=torch.contiguous_format).reshape(1, 1, 1, 64), odd, *want, table, lengths)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


@pytest.mark.parametrize("page", [16, 64])
def test_mass_of_pages_that_sequences_share(pk, page):
    """Twelve sequences with a common prefix: its tokens receive from all of them. A weight is off by at most
    2^-18 and the sums of a few of them by less (the cuts differ with the batch), so 2^-16 in all."""
    shared, own, batch = 4, 2, 12
    cache = pool(shared + own * batch, 2, page, 64)
    table = torch.stack([torch.cat([torch.arange(shared), shared + own * b + torch.arange(own)]) for b in range(batch)])
    table = table.to(torch.int32).to(DEV)
    lengths = torch.tensor([(shared + 1) * page + 1 + b for b in range(batch)], dtype=torch.int32, device=DEV)
    q = torch.randn(batch, 4, 1, 64, device=DEV)
    shape = cache[1].shape + (page,)
    want = torch.zeros(shape, dtype=torch.float64, device=DEV)
    for b in range(batch):
        mass = torch.zeros(shape, device=DEV)
        pk.paged_kv_attention(q[b:b + 1], *cache, table[b:b + 1], lengths[b:b + 1], mass=mass)
        want += mass.double()
    for _ in range(10):
        mass = torch.zeros(shape, device=DEV)
        pk.paged_kv_attention(q, *cache, table, lengths, mass=mass)
        assert ((mass.double() - want).abs() <= 2.0 ** -16 * want).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_nan_query_gives_nothing_to_tokens_it_does_not_see(pk, dtype):
    """Query i of 3 sees all tokens but the last 2 - i."""
    page, n = 16, 44
    cache = pool(3, 1, page, 64)
    table = torch.arange(3, dtype=torch.int32, device=DEV).reshape(1, 3)
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 2, 3, 64, device=DEV).to(dtype)
    for i in range(3):
        bad = q.clone()
        bad[0, 1, i, 7] = float("nan")
        mass = torch.zeros(3, 1, page, device=DEV)
        pk.paged_kv_attention(bad, *cache, table, lengths, mass=mass)
        flat = mass.reshape(-1)
        seen = n - 2 + i
        assert torch.isnan(flat[:seen]).all() and torch.isfinite(flat[seen:n]).all()
        assert (flat[seen:n] > 0).all() and (flat[n:] == 0).all()


@pytest.mark.parametrize("m", [1, 2, 8, 16])
@pytest.mark.parametrize("size,ts", [(1e-33, 1e-4), (1e-36, 3.0), (2e36, 1e-6), (1e-30, 1e-8)])
def test_linear_far_from_one(gv, size, ts, m):
    """fp32 activations whose unit times the tensor scale is subnormal, and sums that pass fp32 before the
    scale: the result is normal and keeps its bits. Bound: as for any linear (a partial sum loses at most
    2^-22 of sum |x| |w|, K / 16 + 64 of them follow one another)."""
    codes, scales = weight(48, 1024, 5)
    scales = (scales.float() * 128).to(E4M3)  # sums of about 2^13 of x's size
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(m, 1024, generator=g, device=DEV) * size
    level = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    level = torch.cat([level, -level])
    w = torch.stack([level[(codes & 15).long()], level[(codes >> 4).long()]], -1).reshape(48, 1024)
    w = w * scales.double().repeat_interleave(16, 1)
    factor = torch.tensor(ts, device=DEV)
    want = x.double() @ w.T * factor.double()
    bound = x.double().abs() @ w.abs().T * factor.double()
    assert 1e-36 < want.abs().median() < 1e38
    y = gv.fp4_w4a16_linear(x, codes, scales, factor)
    assert ((y.double() - want).abs() <= 2.0 ** -24 * want.abs() + (1024 / 16 + 64) * 2.0 ** -22 * bound + 1e-44).all()


def test_linear_many_rows_in_groups(gv):
    """More rows than one group takes: any 32 give what they give alone (fewer alone may be cut along K
    differently)."""
    codes, scales = weight(28672, 2048, 7)
    x = torch.randn(1300, 2048, device=DEV).to(torch.bfloat16)
    bias = torch.randn(28672, device=DEV)
    ts = torch.tensor(0.01, device=DEV)
    y = gv.fp4_w4a16_linear(x, codes, scales, ts, bias)
    for lo in (0, 32, 1120, 1152, 1184, 1268):
        assert torch.equal(y[lo:lo + 32], gv.fp4_w4a16_linear(x[lo:lo + 32], codes, scales, ts, bias))


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attention64(q, cache, table, lengths, causal):
    """(out, received, size, biggest) in 64 bits: size is sum p |v|, biggest a row's largest sum |q| |k| * scale."""
    k_pages, k_scale, v_pages, v_scale = cache
    batch, heads_q, queries, dim = q.shape
    heads, page = k_pages.shape[1:3]
    out, size = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    received, biggest = [], 0.0
    for b, n in enumerate(lengths.tolist()):
        at = table[b, :-(-n // page)].long()
        got = torch.zeros(heads, n, dtype=torch.float64, device=DEV)
        seen = n - queries + 1 + torch.arange(queries, device=DEV) if causal else torch.full((queries,), n, device=DEV)
        hidden = torch.arange(n, device=DEV)[None] >= seen[:, None]
        for h in range(heads if n else 0):
            k, v = ((c[at, h].double() * s[at, h].double()[:, None, None]).reshape(-1, dim)[:n]
                    for c, s in ((k_pages, k_scale), (v_pages, v_scale)))
            for g in range(heads_q // heads):
                x = q[b, h * (heads_q // heads) + g].double() * dim ** -0.5
                p = torch.softmax((x @ k.T).masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
                out[b, h * (heads_q // heads) + g] = p @ v
                size[b, h * (heads_q // heads) + g] = p @ v.abs()
                got[h] += p.sum(0)
                biggest = max(biggest, float((x.abs() @ k.abs().T).max()))
        received.append(got)
    return out, received, size, biggest


def check_attention(pk, q, cache, table, lengths, causal):
    """Bounds: half a unit of the output type; 16-bit queries' weights have 11 bits, fp32 ones' 22; a score is off
    by at most 16 * 2^-22 of the row's largest sum |q| |k| * scale, a weight by twice that; exponentials and
    merges 2^-18. A mass is the sum of its rows' weights, one after the other in fp32."""
    out, received, size, biggest = attention64(q, cache, table, lengths, causal)
    score = 2 * 16 * 2.0 ** -22 * biggest + 2.0 ** -18
    mass = torch.zeros(cache[1].shape + (cache[0].shape[2],), device=DEV)
    got = pk.paged_kv_attention(q, *cache, table, lengths, causal=causal, mass=mass)
    tol = UNIT[q.dtype] * out.abs() + (score + (2.0 ** -20 if q.dtype == torch.float32 else 2.0 ** -11)) * size + 1e-30
    assert ((got.double() - out).abs() <= tol).all()
    page, rows = cache[0].shape[2], q.shape[1] // cache[0].shape[1] * q.shape[2]
    for b, n in enumerate(lengths.tolist()):
        have = mass[table[b, :-(-n // page)].long()].transpose(0, 1).flatten(1)
        want = torch.nn.functional.pad(received[b], (0, have.shape[1] - n))
        assert ((have.double() - want).abs() <= want * (score + (rows + 2) * 2.0 ** -24 + 2.0 ** -20)).all()
    return got


def scratch(pk, q, cache, table, lengths, mass):
    """Bytes that a call takes from the allocator beside its output."""
    pk.paged_kv_attention(q, *cache, table, lengths, mass=mass)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = pk.paged_kv_attention(q, *cache, table, lengths, mass=mass)
    return torch.cuda.max_memory_allocated() - before - out.numel() * out.element_size()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_with_mass(pk, dtype, causal):
    """A prompt whose scores (0.35 GB a sequence) do not fit in what a call takes: its query tokens go in parts."""
    cache = pool(145, 2, 64, 64, 3)
    table = torch.randperm(145, generator=torch.Generator().manual_seed(1))[:144].to(torch.int32).to(DEV)
    table = torch.cat([table[:141], table[141:].repeat(47)]).reshape(2, 141)
    lengths = torch.tensor([9000, 150], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 16, 600, 64, device=DEV).to(dtype)
    check_attention(pk, q, cache, table, lengths, causal)
    mass = torch.zeros(145, 2, 64, device=DEV)
    assert scratch(pk, q, cache, table, lengths, mass) <= 300 << 20


def test_wide_page_table_with_mass(pk):
    """Short sequences in a table with room for 524288 tokens each (64 MB of scores a sequence)."""
    cache = pool(300, 8, 64, 64, 4)
    lengths = torch.tensor([1 + 157 * b for b in range(10)], dtype=torch.int32, device=DEV)
    table = torch.full((10, 8192), -1, dtype=torch.int32, device=DEV)
    table[:, :30] = torch.randperm(300, generator=torch.Generator().manual_seed(2)).reshape(10, 30).to(torch.int32).to(DEV)
    q = torch.randn(10, 32, 1, 64, device=DEV).to(torch.bfloat16)
    wide = check_attention(pk, q, cache, table, lengths, True)
    # the same weights and values, cut differently over the GPU: twice the bound of one of them at most
    narrow = pk.paged_kv_attention(q, *cache, table[:, :30], lengths)
    assert (wide - narrow).abs().max() <= 2.0 ** -6 * narrow.abs().max()
    assert scratch(pk, q, cache, table, lengths, torch.zeros(300, 8, 64, device=DEV)) <= 300 << 20


def test_cache_of_a_large_pool(pk):
    """The class's own table is as wide as the pool; attention and eviction see what is in use, and a prompt
    attends over the paged cache with its mass."""
    cache = pk.PagedFp8KVCache(3, 2, 64, num_pages=4000, page_tokens=64)
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(3, 2, 200, 64, generator=g, device=DEV).to(torch.float16)
    cache.append(x, x * 0.5, counts=[200, 0, 130])
    q = torch.randn(3, 4, 130, 64, generator=g, device=DEV).to(torch.float16)
    out = cache.attend(q)
    parts = cache.k_pages, cache.k_scale, cache.v_pages, cache.v_scale
    assert torch.equal(out, check_attention(pk, q, parts, cache.page_table[:, :4], cache.lengths, True))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    cache.attend(q)
    assert torch.cuda.max_memory_allocated() - before <= 16 << 20
    over, kept = cache.evict(96, recent=32, sinks=4)
    assert over == [0, 2] and cache.lengths.tolist() == cache.tokens == [96, 0, 96]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads_q,queries", [(1, 1), (4, 1), (2, 2), (5, 1), (8, 1), (3, 4), (16, 1), (11, 3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_keep_22_bits(pk, dtype, heads_q, queries, dim):
    """Outputs near zero show what the weights lost: beside the output's own rounding (half a unit) only a score's
    error (twice 16 * 2^-22 of sum |q| |k| * scale, small queries here), 2^-18 for exponentials and merges and
    2^-20 for the weights, of sum p |v|. One, two, four, eight, 12, 16 and 33 rows per KV head."""
    for page, n in ((16, 77), (64, 1500)):
        cache = pool(-(-n // page), 1, page, dim, 11)
        table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV).reshape(1, -1)
        lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(dim + heads_q)
        q = (torch.randn(1, heads_q, queries, dim, generator=g, device=DEV) * 0.05).to(dtype)
        out, _, size, biggest = attention64(q, cache, table, lengths, True)
        tol = UNIT[dtype] * out.abs() + (2 * 16 * 2.0 ** -22 * biggest + 2.0 ** -18 + 2.0 ** -20) * size
        if dtype == torch.float16:
            tol += 2.0 ** -25  # half of its smallest step
        got = pk.paged_kv_attention(q, *cache, table, lengths)
        assert ((got.double() - out).abs() <= tol).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m", [1, 2, 3, 8, 16, 32])
def test_linear_fp32_sums_do_not_drift(gv, m, fmt):
    """Positive products, whose sum only grows: an MMA cuts what it adds to to 24 bits instead of rounding it
    (up to 2^-23 of it, always downwards), so no more than 128 codes' worth, 16 MMAs with x's two terms, may
    follow one another before a rounded addition. The mean over all outputs shows the cuts (up to 16 * 2^-23)
    and leaves the roundings out (2^-24 for what remains of them)."""
    n, k = 8192, 28672  # a warp's part has up to 112 chunks of 256 codes
    g = torch.Generator().manual_seed(m)
    codes = (torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8) & 0x77).to(DEV)
    level = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    w = torch.stack([level[(codes & 15).long()], level[(codes >> 4).long()]], -1).reshape(n, k)
    if fmt == "nvfp4":
        scales = torch.rand(n, k // 16, generator=g).add(0.5).to(E4M3).to(DEV)
        w = w * scales.double().repeat_interleave(16, 1)
    else:
        raw = torch.randint(124, 131, (n, k // 32), generator=g, dtype=torch.int32).to(torch.uint8).to(DEV)
        scales, w = raw.view(torch.float8_e8m0fnu), w * torch.exp2(raw.double() - 127).repeat_interleave(32, 1)
    x = torch.rand(m, k, generator=g).add(0.1).to(DEV)
    want = x.double() @ w.T
    y = gv.fp4_w4a16_linear(x, codes, scales, 1.0, fmt=fmt)
    assert abs(float(((y.double() - want) / want).mean())) <= 16 * 2.0 ** -23 + 2.0 ** -24


@pytest.mark.parametrize("heads_q", [8, 64])
def test_fp32_outputs_do_not_drift(pk, heads_q):
    """Long contexts of positive values: an MMA cuts the sum that it carries (up to 2^-23 of it, always downwards),
    so the products of 16 tokens, two MMAs, are added with a rounding. The mean over a head's outputs shows the
    cuts (2 * 2^-23), exponentials and merges (2^-18) and leaves the roundings out."""
    batch, heads, n, page, dim = 8, 8, 60000, 64, 64
    pages = -(-n // page)
    g = torch.Generator(device=DEV).manual_seed(5)
    codes = [torch.empty(batch * pages, heads, page, dim, dtype=E4M3, device=DEV) for _ in range(2)]
    for c in codes:
        for lo in range(0, batch * pages, 500):
            x = torch.randn(c[lo:lo + 500].shape, generator=g, device=DEV)
            c[lo:lo + 500] = ((x.abs() if c is codes[1] else x) * 64).clamp(-448, 448).to(E4M3)
    scale = torch.full((batch * pages, heads), 2.0 ** -6, device=DEV)
    table = torch.arange(batch * pages, dtype=torch.int32, device=DEV).reshape(batch, pages)
    lengths = torch.full((batch,), n, dtype=torch.int32, device=DEV)
    q = torch.randn(batch, heads_q, dim, generator=g, device=DEV)
    got = pk.paged_kv_attention(q, codes[0], scale, codes[1], scale, table, lengths)
    for b, h in ((0, 0), (3, 5), (7, 7)):
        k, v = ((c[table[b].long(), h].double() * 2.0 ** -6).reshape(-1, dim)[:n] for c in codes)
        rows = slice(h * heads_q // heads, (h + 1) * heads_q // heads)
        want = torch.softmax(q[b, rows].double() @ k.T * dim ** -0.5, -1) @ v
        assert abs(float(((got[b, rows].double() - want) / want).mean())) <= 2 * 2.0 ** -23 + 2.0 ** -18
