"""The paged FP8 KV cache on the GPU: the append and the eviction bit for bit against the numpy
oracle, the attention against its values in 64 bits.

Bounds of the attention, per element, with S = sum p |v| (what roundings of p act on) and B the
largest sum |q| |k| * scale of a row: half a unit of the output type (2^-8, 2^-11 or 2^-24 of
|out|); the weights enter the product with at least 11 significant bits for 16-bit queries (2^-11
of S) and 22 for fp32 ones (2^-20 with the merge's roundings); a score's fp32 sum of D products in
steps of 16 is off by at most 16 * 2^-22 * B, and a weight by twice that, relatively (its own
score and its sum's); exponentials and merges add 2^-18."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import np_bytes, np_values
from oracle import paged_kv as opk

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
KINDS = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def pk():
    from kernel_agent_b200.kernels import paged_kv

    return paged_kv


@pytest.fixture(autouse=True)
def clean_status(request):
    from kernel_agent_b200 import _native as nat

    yield
    assert nat.device_status() == 0


class Cache:
    """A pool on the GPU with its numpy twin; pages in random order, one unused page at least."""

    def __init__(self, lengths, room, heads, page, dim, seed, layout="plain", spare=1):
        g = torch.Generator().manual_seed(seed)
        self.page, self.heads, self.dim = page, heads, dim
        need = [-(-max(n, 1) // page) for n in room]
        order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
        table = torch.full((len(need), max(need)), -7, dtype=torch.int32)  # never read past a sequence's end
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        pages = sum(need) + spare
        x = torch.randn(2, pages, heads, page, dim, generator=g)
        amax = x.abs().amax(dim=(3, 4))
        scale = torch.tensor([[[float(opk.page_scale(v)) for v in r] for r in t] for t in amax.tolist()])
        codes = (x / scale[..., None, None]).to(E4M3)
        mass = torch.rand(pages, heads, page, generator=g)
        if layout == "interleaved":  # K and V of a page side by side, tokens before heads
            pool = codes.view(torch.uint8).permute(1, 0, 3, 2, 4).contiguous().to(DEV).view(E4M3)
            self.k, self.v = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
            both = scale.permute(1, 0, 2).contiguous().to(DEV)
            self.ks, self.vs = both[:, 0], both[:, 1]
            wide = torch.zeros(pages, heads, page + 3)
            wide[..., :page] = mass
            self.mass = wide.to(DEV)[..., :page]
        else:
            self.k, self.v = codes[0].to(DEV), codes[1].to(DEV)
            self.ks, self.vs = scale[0].to(DEV), scale[1].to(DEV)
            self.mass = mass.to(DEV)
        self.table = table.to(DEV)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    @property
    def parts(self):
        return self.k, self.ks, self.v, self.vs

    def np(self):
        return [np_bytes(self.k).copy(), np_values(self.ks).copy(), np_bytes(self.v).copy(),
                np_values(self.vs).copy(), np_values(self.mass).copy()]

    def check(self, want):
        got = self.np()
        for name, a, b in zip(("K", "K scale", "V", "V scale", "mass"), got, want):
            if a.dtype == np.uint8:
                nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
                assert np.all((a == b) | nan), name
            else:
                assert np.array_equal(a, b, equal_nan=True), name


# ------------------------------------------------------------------ append

APPENDS = [  # lengths, counts (None: all), new, kv heads, page, dim
    ([0], None, 1, 1, 16, 64),
    ([0, 5, 16, 63], None, 1, 2, 64, 128),
    ([15, 31, 0], [1, 0, 1], 1, 3, 16, 128),
    ([7, 0, 64, 127], [130, 129, 0, 1], 130, 2, 64, 64),
    ([1], None, 300, 4, 128, 128),
    ([33, 1000], [17, 40], 41, 1, 32, 64),
]


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("case", APPENDS)
def test_append(pk, case, dtype):
    lengths, counts, new, heads, page, dim = case
    used = [new] * len(lengths) if counts is None else counts
    c = Cache(lengths, [a + b for a, b in zip(lengths, used)], heads, page, dim, 3)
    g = torch.Generator().manual_seed(7)
    shape = (len(lengths), heads, new, dim)
    k = (torch.randn(shape, generator=g) * torch.logspace(-3, 3, heads)[:, None, None]).to(dtype).to(DEV)
    v = (torch.randn(shape, generator=g) * 5).to(dtype).to(DEV)
    want = c.np()
    n = opk.append(np_values(k), np_values(v), *want[:4], c.table.cpu().numpy(), lengths, used, want[4])
    got = pk.append_kv_pages(k, v, *c.parts, c.table, c.lengths, mass=c.mass,
                             counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    c.check(want)
    assert got.tolist() == n.tolist() and c.lengths.tolist() == lengths
    again = pk.append_kv_pages(k, v, *c.parts, c.table, c.lengths, mass=c.mass, out_lengths=c.lengths,
                               counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    c.check(want)  # the same tokens in the same slots
    assert again is c.lengths and c.lengths.tolist() == n.tolist()


def test_append_token_by_token(pk):
    """A page grows token by token, loud ones among them, and holds what one append would, up to
    codes that became subnormal."""
    c = Cache([0], [40], 2, 32, 64, 5)
    c.ks.fill_(2.0 ** 90)  # a stale scale of a page that starts empty does not count
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 2, 40, 64, generator=g) * torch.exp(torch.randn(1, 2, 40, 1, generator=g))
    want = c.np()
    for t in range(40):
        xt = x[:, :, t:t + 1].to(torch.bfloat16).to(DEV)
        n = opk.append(np_values(xt), np_values(xt), *want[:4], c.table.cpu().numpy(), [t], None, want[4])
        pk.append_kv_pages(xt, xt, *c.parts, c.table, c.lengths, mass=c.mass, out_lengths=c.lengths)
    c.check(want)
    assert c.lengths.tolist() == n.tolist() == [40]
    xs = x.to(torch.bfloat16).to(DEV)
    one = Cache([0], [40], 2, 32, 64, 5)
    pk.append_kv_pages(xs, xs, *one.parts, one.table, one.lengths)
    used = c.table[0, :2].cpu().numpy()
    assert np.array_equal(np_values(c.ks)[used], np_values(one.ks)[used])


@pytest.mark.parametrize("held", [0, 3])
def test_append_special_values(pk, held):
    """Zeros, infinities, NaN, the smallest and the largest fp32 values; old scales that are no
    powers of two."""
    for fill in ("zero", "inf", "nan", "tiny", "huge", "448", "449"):
        c = Cache([held], [20], 1, 16, 64, 11)
        c.ks.mul_(1.5)
        c.vs.fill_(3e-39 if fill == "tiny" else 0.3)
        x = torch.zeros(1, 1, 17, 64)
        if fill == "inf":
            x[0, 0, 2, 5], x[0, 0, 4, 6], x[0, 0, 4, 7] = float("inf"), float("-inf"), 2.0
        elif fill == "nan":
            x[0, 0, 1, :], x[0, 0, 1, 9] = float("nan"), 1e-3
        elif fill == "tiny":
            x[0, 0, :, 0], x[0, 0, 5, 1] = 1e-45, 1e-38
        elif fill == "huge":
            x[0, 0, :, 0], x[0, 0, 3, 3] = 3.4e38, -1.0
        elif fill != "zero":
            x += float(fill)
        want = c.np()
        opk.append(x.numpy(), x.numpy() * 0.5, *want[:4], c.table.cpu().numpy(), [held], None, want[4])
        pk.append_kv_pages(x.to(DEV), (x * 0.5).to(DEV), *c.parts, c.table, c.lengths, mass=c.mass)
        c.check(want)


def test_append_strided(pk):
    """Tokens before heads, K and V in one projection's output, an interleaved pool."""
    c = Cache([9, 0], [60, 51], 3, 32, 64, 13, layout="interleaved")
    qkv = torch.randn(2, 51, 2, 3, 64, device=DEV).to(torch.bfloat16)
    k, v = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    want = c.np()
    opk.append(np_values(k), np_values(v), *want[:4], c.table.cpu().numpy(), [9, 0], None, want[4])
    pk.append_kv_pages(k, v, *c.parts, c.table, c.lengths, mass=c.mass)
    c.check(want)


# ------------------------------------------------------------------ attention

ATTENDS = [  # lengths, query tokens, query heads, kv heads, page, dim, causal
    ([1], 1, 1, 1, 16, 64, True),
    ([0, 1, 2, 16, 17, 333], 1, 8, 2, 16, 128, True),
    ([5, 0, 3, 64], 4, 6, 2, 32, 64, True),
    ([5, 0, 3, 64], 4, 6, 2, 32, 64, False),
    ([1000, 7, 257], 1, 32, 8, 64, 128, True),
    ([4097], 2, 5, 1, 128, 128, True),
    ([130, 31], 3, 21, 1, 64, 64, True),   # 63 rows of one KV head
    ([700] * 40, 1, 8, 8, 16, 64, True),
    ([20000, 1, 3], 1, 4, 4, 64, 128, True),
]


def bounds(q, c, lengths, out, size, scale, dtype):
    biggest = np.zeros(q.shape[:3])
    hq, heads = q.shape[1], c.heads
    for b, n in enumerate(lengths):
        if n:
            k = np.abs(opk.values(np_bytes(c.k), np_values(c.ks), c.table.cpu().numpy()[b], n))
            for h in range(hq):
                biggest[b, h] = (np.abs(q[b, h]).astype(np.float64) @ k[h // (hq // heads)].T).max(-1) * scale
    score = 2 * 16 * 2.0 ** -22 * biggest[..., None] + 2.0 ** -18
    return UNIT[dtype] * np.abs(out) + (score + (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -11)) * size + 1e-30, score


@pytest.mark.parametrize("layout", ["plain", "interleaved"])
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("case", ATTENDS)
def test_attention(pk, case, dtype, layout):
    lengths, lq, hq, heads, page, dim, causal = case
    c = Cache(lengths, lengths, heads, page, dim, 21, layout)
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(len(lengths), hq, lq, dim, generator=g) * 1.5).to(dtype).to(DEV)
    scale = None if dim == 64 else 0.11
    want, received, size = opk.attention(np_values(q), *c.np()[:4], c.table.cpu().numpy(), lengths, scale, causal)
    tol, score = bounds(np_values(q), c, lengths, want, size, dim ** -0.5 if scale is None else scale, dtype)
    before = c.np()[4]
    got = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths, scale=scale, causal=causal, mass=c.mass)
    assert got.dtype == dtype and got.shape == q.shape
    assert np.all(np.abs(np_values(got) - want) <= tol)
    after, used = c.np()[4], np.zeros(before.shape, bool)
    table = c.table.cpu().numpy()
    for b, n in enumerate(lengths):
        for t0 in range(0, n, page):
            t1, p = min(n, t0 + page), table[b, t0 // page]
            gain = after[p, :, :t1 - t0].astype(np.float64) - before[p, :, :t1 - t0]
            add = received[b][:, t0:t1]
            assert np.all(np.abs(gain - add) <= add * (score[b].max() + 2.0 ** -20) + 2.0 ** -23 * (before[p, :, :t1 - t0] + add))
            used[p, :, :t1 - t0] = True
    assert np.array_equal(after[~used], before[~used])
    plain = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths, scale=scale, causal=causal)
    assert np.all(np.abs(np_values(plain) - want) <= tol)
    if lq == 1:
        flat = pk.paged_kv_attention(q[:, :, 0], *c.parts, c.table, c.lengths, scale=scale, causal=causal)
        assert torch.equal(flat, plain[:, :, 0])


@pytest.mark.parametrize("dtype", KINDS)
def test_attention_scales(pk, dtype):
    """Scales far apart, no powers of two, zero (a page of zeros whatever its codes), and queries
    far from 1: pages weigh by their values, not by their codes."""
    c = Cache([200], [200], 2, 16, 64, 31)
    pages = c.ks.shape[0]
    c.ks.copy_(c.ks * torch.logspace(-1, 0.5, pages, device=DEV)[:, None])
    c.vs.copy_(c.vs * torch.logspace(-12, 12, pages, device=DEV)[:, None] * 1.7)
    c.vs[c.table[0, 3].long()] = 0.0
    c.ks[c.table[0, 5].long()] = 0.0
    q = (torch.randn(1, 6, 1, 64) * torch.logspace(-3, 0, 6)[:, None, None]).to(dtype).to(DEV)
    want, _, size = opk.attention(np_values(q), *c.np()[:4], c.table.cpu().numpy(), [200])
    tol, _ = bounds(np_values(q), c, [200], want, size, 0.125, dtype)
    got = np_values(pk.paged_kv_attention(q, *c.parts, c.table, c.lengths)) if dtype != torch.float16 else None
    if got is not None:  # fp16 outputs would overflow
        assert np.all(np.abs(got - want) <= tol)
    big = (q.float() * 1e30).to(dtype) if dtype != torch.float16 else q * 64.0  # |q| up to fp16's range
    s = 0.125 / (1e30 if dtype != torch.float16 else 64.0)
    c.vs.fill_(0.25)
    want, _, size = opk.attention(np_values(big), *c.np()[:4], c.table.cpu().numpy(), [200], s)
    tol, _ = bounds(np_values(big), c, [200], want, size, s, dtype)
    got = np_values(pk.paged_kv_attention(big, *c.parts, c.table, c.lengths, scale=s))
    assert np.all(np.abs(got - want) <= tol)


def test_attention_ignores_what_is_not_cached(pk):
    """NaN codes and scales in slots and pages past a sequence's end change nothing."""
    lengths = [37, 0, 64]
    c = Cache(lengths, lengths, 2, 32, 128, 41)
    q = torch.randn(3, 4, 2, 128, device=DEV).to(torch.bfloat16)
    clean = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths)
    for b, n in enumerate(lengths):
        if n % 32:
            page = int(c.table[b, n // 32])
            c.k.view(torch.uint8)[page, :, n % 32:] = 0x7F
            c.v.view(torch.uint8)[page, :, n % 32:] = 0xFF
    for page in [int(c.table[1, 0]), *c.free.tolist()]:
        c.ks[page], c.vs[page] = float("nan"), float("inf")
        c.k.view(torch.uint8)[page] = 0x7F
    assert torch.equal(pk.paged_kv_attention(q, *c.parts, c.table, c.lengths), clean)
    assert torch.count_nonzero(clean[1]) == 0


def test_attention_nan_and_inf(pk):
    """A NaN key reaches the queries that see it and no others; an infinite query gives NaN."""
    c = Cache([40], [40], 1, 16, 64, 43)
    q = torch.randn(1, 2, 3, 64, device=DEV)
    c.k.view(torch.uint8)[int(c.table[0, 2]), 0, 7, 3] = 0x7F  # token 39: only the last query sees it
    got = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths)
    assert torch.isfinite(got[:, :, :2]).all() and torch.isnan(got[:, :, 2]).all()
    c = Cache([40], [40], 1, 16, 64, 44)
    q[0, 1, 0, 5] = float("inf")
    got = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths)
    assert torch.isnan(got[0, 1, 0]).all() and torch.isfinite(got[0, 0]).all() and torch.isfinite(got[0, 1, 1:]).all()


def test_attention_far_offsets(pk):
    """Pages past 2^31 and 2^32 bytes of the pool."""
    pages, heads, page, dim = 40000, 8, 128, 128  # 5.2 GB each
    k = torch.empty(pages, heads, page, dim, dtype=E4M3, device=DEV)
    v = torch.empty(pages, heads, page, dim, dtype=E4M3, device=DEV)
    ks, vs = torch.ones(pages, heads, device=DEV), torch.ones(pages, heads, device=DEV)
    mass = torch.zeros(pages, heads, page, device=DEV)
    at = [5, 20000, pages - 1]
    table = torch.tensor([at], dtype=torch.int32, device=DEV)
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    small = Cache([0], [300], heads, page, dim, 51, spare=3)
    x = torch.randn(2, 1, heads, 300, dim, device=DEV).to(torch.bfloat16)
    q = torch.randn(1, 16, 1, dim, device=DEV).to(torch.bfloat16)
    n = pk.append_kv_pages(x[0], x[1], k, ks, v, vs, table, lengths, mass=mass)
    m = pk.append_kv_pages(x[0], x[1], *small.parts, small.table, small.lengths, mass=small.mass)
    a = pk.paged_kv_attention(q, k, ks, v, vs, table, n, mass=mass)
    b = pk.paged_kv_attention(q, *small.parts, small.table, m, mass=small.mass)
    assert torch.equal(a, b)
    to = torch.tensor([[pages - 2, 30000]], dtype=torch.int32, device=DEV)
    kept, n2 = pk.evict_kv_pages(k, ks, v, vs, mass, table, n, to, budget=200, recent=10)
    to_small = small.free[:2].reshape(1, 2).to(DEV)
    kept2, m2 = pk.evict_kv_pages(*small.parts, small.mass, small.table, m, to_small, budget=200, recent=10)
    assert torch.equal(kept, kept2) and n2.tolist() == m2.tolist() == [200]
    assert torch.equal(pk.paged_kv_attention(q, k, ks, v, vs, to, n2),
                       pk.paged_kv_attention(q, *small.parts, to_small, m2))


def test_streams_graphs_and_repeats(pk):
    """The same answers on another stream, replayed from a graph, and every time."""
    lengths = [513, 64, 2000, 1]
    c = Cache(lengths, [n + 8 for n in lengths], 2, 64, 128, 61)
    q = torch.randn(4, 8, 1, 128, device=DEV).to(torch.bfloat16)
    k = torch.randn(4, 2, 1, 128, device=DEV).to(torch.bfloat16)

    def step():
        pk.append_kv_pages(k, k, *c.parts, c.table, c.lengths, mass=c.mass, out_lengths=c.lengths)
        return pk.paged_kv_attention(q, *c.parts, c.table, c.lengths, mass=c.mass)

    start = [t.clone() for t in (c.k, c.ks, c.v, c.vs, c.mass, c.lengths)]

    def reset():
        for t, s in zip((c.k, c.ks, c.v, c.vs, c.mass, c.lengths), start):
            t.copy_(s)

    want = [step().clone() for _ in range(3)]
    state = [t.clone() for t in (c.k, c.mass, c.lengths)]
    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step().clone() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    reset()
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    for t, s in zip((c.k, c.mass, c.lengths), state):
        assert torch.equal(t.view(torch.uint8), s.view(torch.uint8))


# ------------------------------------------------------------------ evict

EVICTS = [  # lengths, kv heads, page, dim, budget, recent, sinks
    ([100], 1, 16, 64, 40, 10, 2),
    ([0, 1, 39, 40, 41, 300], 2, 32, 128, 40, 8, 4),
    ([257, 1000], 3, 64, 64, 256, 0, 0),
    ([500], 2, 128, 128, 1, 0, 0),
    ([500], 2, 128, 128, 1, 1, 0),
    ([500, 77], 1, 16, 128, 64, 60, 4),
    ([5000, 3], 8, 64, 128, 600, 100, 1),
    ([40000], 2, 64, 64, 3999, 1, 0),
    ([70000], 1, 64, 64, 69999, 5, 5),
]


@pytest.mark.parametrize("kind", ["random", "ties", "special"])
@pytest.mark.parametrize("case", EVICTS)
def test_evict(pk, case, kind):
    lengths, heads, page, dim, budget, recent, sinks = case
    width = -(-budget // page)
    c = Cache(lengths, lengths, heads, page, dim, 71, spare=len(lengths) * width,
              layout="interleaved" if kind == "ties" else "plain")
    g = torch.Generator(device=DEV).manual_seed(5)
    if kind == "ties":
        c.mass.copy_(torch.randint(0, 3, c.mass.shape, generator=g, device=DEV).float() - 1.0)
        c.mass[c.mass == 0] = -0.0
    elif kind == "special":
        c.mass.copy_(torch.randn(c.mass.shape, generator=g, device=DEV))
        odd = torch.randint(0, 30, c.mass.shape, generator=g, device=DEV)
        for i, v in enumerate((float("nan"), float("inf"), float("-inf"), 1e-45, -0.0, 0.0)):
            c.mass[odd == i] = v
        c.ks.mul_(torch.logspace(-3, 3, c.ks.shape[0], device=DEV)[:, None])
        c.k.view(torch.uint8)[:, :, 3, 2] = 0x7F
    to = c.free.reshape(len(lengths), width)
    want = c.np()
    kept, n = opk.evict(*want, c.table.cpu().numpy(), lengths, to.numpy(), budget, recent, sinks)
    got, m = pk.evict_kv_pages(*c.parts, c.mass, c.table, c.lengths, to.to(DEV), budget=budget, recent=recent,
                               sinks=sinks)
    assert np.array_equal(got.cpu().numpy(), kept) and m.tolist() == n.tolist()
    c.check(want)


def test_evicted_cache_attends(pk):
    """What was heavy stays: dropping tokens that received next to nothing changes little."""
    c = Cache([600], [600], 2, 32, 64, 81, spare=4)
    c.mass.zero_()
    q = torch.randn(1, 4, 1, 64, device=DEV) * 6.0
    full = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths, mass=c.mass)
    table = c.table[0].long()
    held = c.mass[table].transpose(0, 1).reshape(2, -1)[:, :600]
    kept, n = pk.evict_kv_pages(*c.parts, c.mass, c.table, c.lengths, c.free.reshape(1, 4).to(DEV), budget=128)
    lost = 2.0 - held.gather(1, kept[0].long()).sum(1)  # of two query heads per KV head
    part = pk.paged_kv_attention(q, *c.parts, c.free.reshape(1, 4).to(DEV), n)
    biggest = float((c.v.float() * c.vs[..., None, None]).abs().max())
    for h in range(4):
        assert float((part - full)[0, h].abs().max()) <= 2.0 * float(lost[h // 2]) * biggest + 1e-4 * biggest


# ------------------------------------------------------------------ errors


def test_bad_numbers_raise_the_status(pk):
    """Page numbers outside the pool and lengths past the table are skipped and reported."""
    from kernel_agent_b200 import _native as nat

    c = Cache([20, 20], [40, 40], 1, 16, 64, 91)
    x = torch.ones(2, 1, 3, 64, device=DEV)
    q = torch.randn(2, 2, 1, 64, device=DEV)
    good = pk.paged_kv_attention(q, *c.parts, c.table, c.lengths)
    bad = c.table.clone()
    bad[1, 0], bad[1, 1] = 1 << 20, -3
    got = pk.paged_kv_attention(q, *c.parts, bad, c.lengths)
    assert torch.equal(got[0], good[0])
    assert nat.device_status() == 2
    before = c.np()
    pk.append_kv_pages(x[1:], x[1:], *c.parts, bad[1:], c.lengths[1:])
    assert nat.device_status() == 2
    c.check(before)
    long = torch.tensor([20, 49], dtype=torch.int32, device=DEV)
    n = pk.append_kv_pages(x, x, *c.parts, c.table, long, mass=c.mass)
    assert nat.device_status() == 2 and n.tolist() == [23, 48]
    got = pk.paged_kv_attention(q, *c.parts, c.table, long)
    assert nat.device_status() == 2 and torch.isfinite(got).all()
    minus = torch.tensor([-1, 20], dtype=torch.int32, device=DEV)
    assert torch.count_nonzero(pk.paged_kv_attention(q, *c.parts, c.table, minus)[0]) == 0
    assert nat.device_status() == 2
    kept, n = pk.evict_kv_pages(*c.parts, c.mass, bad, c.lengths, c.free.reshape(1, 1).expand(2, 1).to(DEV), budget=8)
    assert nat.device_status() == 2 and n.tolist() == [8, 8]


def test_refusals(pk):
    c = Cache([20], [40], 2, 16, 64, 95)
    x = torch.ones(1, 2, 3, 64, device=DEV)
    q = torch.ones(1, 4, 1, 64, device=DEV)
    parts = list(c.parts)

    def swap(i, t):
        return [t if j == i else p for j, p in enumerate(parts)]

    with pytest.raises(ValueError, match="CUDA tensor"):
        pk.append_kv_pages(x.cpu(), x, *parts, c.table, c.lengths)
    for bad in (swap(0, c.k[:, :, :12]), swap(0, c.k.float()), swap(1, c.ks.double()), swap(3, c.vs[:, :1])):
        with pytest.raises(ValueError):
            pk.append_kv_pages(x, x, *bad, c.table, c.lengths)
        with pytest.raises(ValueError):
            pk.paged_kv_attention(q, *bad, c.table, c.lengths)
    with pytest.raises(ValueError, match="page_tokens"):
        pk.paged_kv_attention(q, c.k.repeat(1, 1, 3, 1), c.ks, c.v.repeat(1, 1, 3, 1), c.vs, c.table, c.lengths)
    with pytest.raises(ValueError, match="page_table"):
        pk.paged_kv_attention(q, *parts, c.table.long(), c.lengths)
    with pytest.raises(ValueError, match="lengths"):
        pk.paged_kv_attention(q, *parts, c.table, c.lengths.long())
    with pytest.raises(ValueError, match="fit"):
        pk.paged_kv_attention(q[:, :3], *parts, c.table, c.lengths)
    with pytest.raises(ValueError, match="q must be"):
        pk.paged_kv_attention(q[0, 0], *parts, c.table, c.lengths)
    with pytest.raises(ValueError, match="dtype"):
        pk.paged_kv_attention(q.double(), *parts, c.table, c.lengths)
    with pytest.raises(ValueError, match="out must"):
        pk.paged_kv_attention(q, *parts, c.table, c.lengths, out=q.half())
    with pytest.raises(ValueError, match="aligned"):
        paged = torch.empty(q.numel() + 1, device=DEV)[1:].reshape(q.shape)
        pk.paged_kv_attention(q, *parts, c.table, c.lengths, out=paged)
    with pytest.raises(ValueError, match="expected k and v"):
        pk.append_kv_pages(x[:, :1], x[:, :1], *parts, c.table, c.lengths)
    with pytest.raises(ValueError, match="both be"):
        pk.append_kv_pages(x, x.half(), *parts, c.table, c.lengths)
    with pytest.raises(ValueError, match="counts"):
        pk.append_kv_pages(x, x, *parts, c.table, c.lengths, counts=c.lengths.long())
    to = c.free.reshape(1, 1).to(DEV)
    for kw in ({"budget": 0}, {"budget": 8, "recent": 9}, {"budget": 8, "recent": 6, "sinks": 3}, {"budget": 8, "recent": -1}):
        with pytest.raises(ValueError, match="budget"):
            pk.evict_kv_pages(*parts, c.mass, c.table, c.lengths, to, **kw)
    with pytest.raises(ValueError, match="out_page_table"):
        pk.evict_kv_pages(*parts, c.mass, c.table, c.lengths, to, budget=17)
    with pytest.raises(ValueError, match="other pages"):
        pk.evict_kv_pages(*parts, c.mass, c.table, c.lengths, c.table, budget=17)
    with pytest.raises(ValueError, match="mass"):
        pk.evict_kv_pages(*parts, None, c.table, c.lengths, to, budget=8)
    empty = pk.append_kv_pages(x[:, :, :0], x[:, :, :0], *parts, c.table, c.lengths)
    assert empty.tolist() == [20]
    assert pk.paged_kv_attention(q[:, :, :0], *parts, c.table, c.lengths).shape == (1, 4, 0, 64)
