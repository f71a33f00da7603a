"""Host side of the decode operators without a GPU: what a wrapper hands to the C entry points, with
the entry point itself replaced and the tensors on the CPU."""

from __future__ import annotations

import ctypes
import threading
from types import SimpleNamespace

import pytest
import torch

from kernel_agent_b200 import _native as nat
from kernel_agent_b200.kernels import _launch, gemv, paged_kv

pytestmark = pytest.mark.skipif(not nat.LIB_PATH.exists(), reason="libkab.so is not built")


@pytest.fixture
def calls(monkeypatch):
    """The wrappers on CPU tensors: every entry point but the workspace queries is recorded as
    ``(name, args)`` and handed to ``calls.seen`` where that is set."""
    log = SimpleNamespace(made=[], seen=None)

    def call(name, device, *args):
        if name == "kab_gemv_fp4_workspace":
            return nat.call(name, *args)
        if name == "kab_kv_pages_attention_workspace":  # the real one asks the GPU for its resident blocks
            args[1]._obj.value = 256
            return
        log.made.append((name, args))
        if log.seen is not None:
            log.seen(name, args)

    for module in (gemv, paged_kv):
        monkeypatch.setattr(module, "call", call)
        monkeypatch.setattr(module, "device_of", lambda *tensors: -1)  # as Tensor.get_device() says on the CPU
        monkeypatch.setattr(module, "stream_of", lambda device: 0)
    monkeypatch.setattr(_launch, "torch", SimpleNamespace(
        empty=torch.empty, uint8=torch.uint8, device=lambda *a: torch.device("cpu"),
        _C=SimpleNamespace(_cuda_isCurrentStreamCapturing=lambda: False)))
    return log


def test_calls_of_two_threads_have_scratch_of_their_own(calls):
    """A call enqueues several launches that pass data through its scratch memory, and the interpreter runs
    other threads meanwhile: two calls on one stream must not share it."""
    x = torch.zeros(5, 8192, dtype=torch.bfloat16)
    codes, scales = torch.zeros(64, 4096, dtype=torch.uint8), torch.zeros(64, 512, dtype=torch.uint8)
    spans = []
    inside = threading.Barrier(2, timeout=20)

    def seen(name, args):
        spans.append((args[-3], args[-3] + args[-2]))
        inside.wait()  # both calls are between their launches

    calls.seen = seen
    run = lambda: gemv.fp4_w4a16_linear(x, codes, scales, 1.0)  # noqa: E731
    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    (a0, a1), (b0, b1) = spans
    assert a1 > a0 and b1 > b0
    assert a1 <= b0 or b1 <= a0


@pytest.fixture
def host_cache(monkeypatch):
    """``PagedFp8KVCache`` with its tensors on the CPU (its functions replaced by a test where it calls them)."""

    class Cpu:
        def __getattr__(self, name):
            return getattr(torch, name)

        def device(self, *_):
            return SimpleNamespace(type="cuda")

        def zeros(self, *shape, device=None, **kw):
            return torch.zeros(*shape, **kw)

        def ones(self, *shape, device=None, **kw):
            return torch.ones(*shape, **kw)

        def full(self, *args, device=None, **kw):
            return torch.full(*args, **kw)

        cuda = SimpleNamespace(is_current_stream_capturing=lambda: False)

    monkeypatch.setattr(paged_kv, "torch", Cpu())
    monkeypatch.setattr(paged_kv, "to_device", lambda values, dtype, device: torch.tensor(values, dtype=dtype))
    return lambda *args, **kw: paged_kv.PagedFp8KVCache(*args, device="cuda", **kw)


def test_page_table_names_only_pages_of_the_sequence(host_cache):
    """Entries past a sequence's pages are outside the pool, so that a kernel that reads one reports it instead
    of touching another sequence's page."""
    cache = host_cache(3, 1, 64, num_pages=10, page_tokens=16, max_pages=6)
    assert (cache.page_table == -1).all()
    cache.reserve([33, 0, 16])
    table = cache.page_table.tolist()
    assert [sum(p >= 0 for p in row) for row in table] == [3, 0, 1]
    assert table[0][3:] == [-1] * 3 and table[1] == [-1] * 6 and table[2][1:] == [-1] * 5
    cache.free(0)
    assert cache.page_table[0].tolist() == [-1] * 6 and cache.page_table[2].tolist() == table[2]


def test_captured_steps_are_counted(host_cache):
    """Tokens that replays appended are made known with advance(): the next reservation goes by them, and
    no more can be counted than pages were reserved for."""
    cache = host_cache(2, 1, 64, num_pages=10, page_tokens=16)
    cache.reserve([40, 16])
    assert cache.tokens == [0, 0]
    cache.advance([40, 16])
    assert cache.tokens == [40, 16] and [len(p) for p in cache._pages] == [3, 1]
    cache.reserve([9, 1])
    assert [len(p) for p in cache._pages] == [4, 2]
    assert (cache.page_table >= 0).sum(1).tolist() == [4, 2]
    with pytest.raises(ValueError, match="reserve"):
        cache.advance([25, 0])
    with pytest.raises(ValueError, match="counts"):
        cache.advance([1])
    with pytest.raises(ValueError, match="counts"):
        cache.advance([1, -1])
    assert cache.tokens == [40, 16]


def test_no_table_is_written_inside_a_capture(host_cache, monkeypatch):
    """A captured copy of host page numbers would be replayed from host memory that is gone by then."""
    cache = host_cache(1, 1, 64, num_pages=8, page_tokens=16)
    cache.reserve([40])
    cache.advance([40])
    pages, free, table = list(cache._pages[0]), list(cache._free), cache.page_table.clone()
    monkeypatch.setattr(paged_kv.torch.cuda, "is_current_stream_capturing", lambda: True)
    for method, args in ((cache.reserve, ([20],)), (cache.evict, (16,)), (cache.free, (0,))):
        with pytest.raises(RuntimeError, match="reserve"):
            method(*args)
        assert cache._pages == [pages] and cache._free == free and cache.tokens == [40]
        assert torch.equal(cache.page_table, table)
    cache.reserve([1])  # no page needed: nothing is written


def test_a_failed_eviction_keeps_the_free_pages(host_cache, monkeypatch):
    cache = host_cache(1, 1, 64, num_pages=8, page_tokens=16)
    cache.reserve([40])
    cache.advance([40])
    before = list(cache._free)

    def fail(*args, **kw):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(paged_kv, "evict_kv_pages", fail)
    with pytest.raises(RuntimeError, match="memory"):
        cache.evict(20)
    assert cache._free == before and cache.tokens == [40] and len(cache._pages[0]) == 3


def misaligned(shape, dtype=torch.bfloat16):
    """A contiguous tensor one element past a 16-byte boundary."""
    flat = torch.arange(17 + torch.Size(shape).numel(), dtype=torch.float32).to(dtype)
    start = (16 - flat.data_ptr() % 16) % 16 // flat.element_size() + 1
    return flat[start:start + torch.Size(shape).numel()].view(shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 3])
def test_linear_takes_x_off_16_bytes(calls, m, dtype):
    x = misaligned((m, 64), dtype)
    assert x.is_contiguous() and x.data_ptr() % 16
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    gemv.fp4_w4a16_linear(x, codes, scales, 1.0)
    (name, args), = calls.made
    assert name == "kab_gemv_fp4" and args[0] % 16 == 0 and args[2] % 8 == 0


def cpu_pool(pages=4, heads=1, page=16, dim=64):
    codes = torch.zeros(pages, heads, page, dim, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return codes, torch.ones(pages, heads), codes.clone(), torch.ones(pages, heads)


def test_append_takes_rows_off_16_bytes(calls):
    """Contiguous keys and values that start anywhere, and size-1 dimensions of any stride."""
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    off = misaligned((1, 1, 3, 64))
    odd = torch.zeros(1, 1, 2, 70, dtype=torch.bfloat16)[:, :, 1:, :64].as_strided((1, 1, 1, 64), (70, 35, 70, 1), 0)
    assert odd.is_contiguous() and off.is_contiguous() and off.data_ptr() % 16
    for x in (off, odd):
        calls.made.clear()
        paged_kv.append_kv_pages(x, x, *cpu_pool(), table, lengths)
        (name, args), = calls.made
        assert name == "kab_kv_pages_append" and args[1] % 16 == args[2] % 16 == 0
        assert all(s % 8 == 0 for s in args[4:10])


def attend(q, scale=None, heads=1, mass=None):
    table, lengths = torch.zeros(q.shape[0], 4, dtype=torch.int32), torch.zeros(q.shape[0], dtype=torch.int32)
    return paged_kv.paged_kv_attention(q, *cpu_pool(heads=heads), table, lengths, scale=scale, mass=mass)


def test_attention_reads_its_scale_every_call(calls):
    """A scale held in a tensor that changes between calls."""
    scale = torch.tensor(0.5)
    q = torch.zeros(1, 2, 1, 64)
    attend(q, scale)
    scale.fill_(0.25)
    attend(q, scale)
    assert [args[0]._obj.sm_scale for _, args in calls.made] == [0.5, 0.25]


def test_what_is_kept_for_layouts_is_bounded(calls):
    """Shapes that change from step to step (rows, table widths) do not grow the wrappers' tables without end."""
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    for m in range(1, 1200):
        gemv.fp4_w4a16_linear(torch.zeros(m, 64), codes, scales, 1.0)
        attend(torch.zeros(1, 1, 1, 64), 1.0 / m)
    assert len(gemv._PLANS) <= 1024 and len(paged_kv._TEMPLATES) <= 1024


def test_a_pool_without_heads_is_refused(calls):
    with pytest.raises(ValueError, match="KV head"):
        attend(torch.zeros(1, 2, 1, 64), heads=0)


def test_pool_strides_of_single_rows_do_not_count(calls):
    """A pool of one head, or one page, whose stride along it is anything."""
    flat = torch.zeros(4 * 16 * 64 + 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    pages = flat.as_strided((4, 1, 16, 64), (1024, 7, 64, 1))
    one = flat.as_strided((1, 2, 16, 64), (1 << 33, 1024, 64, 1))
    for codes, heads in ((pages, 1), (one, 2)):
        scale = torch.ones(codes.shape[:2])
        table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
        calls.made.clear()
        paged_kv.paged_kv_attention(torch.zeros(1, 2, 1, 64), codes, scale, codes, scale, table, lengths)
        cache = calls.made[0][1][0]._obj.cache
        assert cache.k_stride_head % 16 == cache.v_stride_head % 16 == 0
        assert cache.k_stride_page < 1 << 31 and cache.v_stride_page < 1 << 31


@pytest.mark.parametrize("m,n,k", [(2048, 28672, 8192), (65535, 57344, 8192), (1171, 28672, 2048), (4000, 4096, 131072)])
@pytest.mark.parametrize("fmt", [nat.KAB_NVFP4, nat.KAB_MXFP4])
def test_linear_workspace_is_bounded(m, n, k, fmt):
    """Many rows go through in groups: 256 MB of scratch, or what 32 rows need where that is more."""
    def size(rows):
        found = ctypes.c_size_t(0)
        nat.call("kab_gemv_fp4_workspace", rows, n, k, fmt, nat.KAB_BF16, ctypes.byref(found))
        return found.value

    assert size(m) <= max(256 << 20, size(32))
    for rows in (1, 2, 5, 8, 9, 16, 17, 31):  # what is left for the last group needs no more
        assert size(m // 32 * 32 + rows) <= max(256 << 20, size(32), size(rows))


def test_the_cache_hands_over_only_the_table_in_use(host_cache, monkeypatch):
    """The launches and scratch memory of attention and eviction follow the table's width, by default that of
    the whole pool: they get as much of it as a sequence holds pages."""
    seen = []
    monkeypatch.setattr(paged_kv, "paged_kv_attention", lambda q, k, ks, v, vs, table, lengths, **kw: seen.append(table.clone()))

    def evict(k, ks, v, vs, mass, table, lengths, to, budget, **kw):
        seen.append(table.clone())
        return torch.zeros(len(lengths), 1, budget, dtype=torch.int32), torch.full_like(lengths, budget)

    monkeypatch.setattr(paged_kv, "evict_kv_pages", evict)
    cache = host_cache(3, 1, 64, num_pages=400, page_tokens=16)
    q = torch.zeros(3, 1, 64)
    cache.attend(q)
    cache.reserve([5, 60, 17])
    cache.attend(q)
    cache.advance([5, 60, 17])
    cache.evict(20)
    assert [tuple(t.shape) for t in seen] == [(3, 1), (3, 4), (1, 4)]
    assert seen[2][0].tolist() == seen[1][1].tolist()


def test_a_page_taken_writes_its_table_entry_alone(host_cache, monkeypatch):
    """A step that takes a page sends that entry, not the whole table; entries of freed and moved pages go."""
    sent = []

    def to_device(values, dtype, device):
        t = torch.tensor(values, dtype=dtype)
        sent.append(t.numel())
        return t

    monkeypatch.setattr(paged_kv, "to_device", to_device)
    monkeypatch.setattr(paged_kv, "evict_kv_pages", lambda k, ks, v, vs, mass, table, lengths, to, budget, **kw: (
        torch.zeros(len(lengths), 1, budget, dtype=torch.int32), torch.full_like(lengths, budget)))
    cache = host_cache(8, 1, 64, num_pages=1000, page_tokens=16)

    def check():
        want = torch.full((8, 1000), -1, dtype=torch.int32)
        for b, pages in enumerate(cache._pages):
            want[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        assert torch.equal(cache.page_table, want)

    for counts in ([100, 0, 16, 1, 30, 2, 2, 2], [0] * 7 + [20], [16] * 8):
        sent.clear()
        cache.reserve(counts)
        cache.advance(counts)
        check()
        assert sum(sent) <= 100
    sent.clear()
    over, _ = cache.evict(20)
    assert over == [0, 2, 4, 7]
    check()
    cache.free(1)
    check()
    cache.free(1)
    check()
    assert sum(sent) <= 100


def test_eviction_refuses_to_overwrite_the_lengths_it_reads():
    """Blocks read a sequence's length while the first one writes the new one."""
    p = nat.KabKvPages()
    p.k_pages = p.v_pages = p.k_scale = p.v_scale = p.mass = p.page_table = p.lengths = 256
    p.num_pages, p.heads_kv, p.page_tokens, p.head_dim, p.max_pages, p.batch, p.table_stride = 8, 2, 64, 128, 4, 1, 4
    p.k_stride_page = p.v_stride_page = 2 * 64 * 128
    p.k_stride_head = p.v_stride_head = 64 * 128
    p.k_stride_token = p.v_stride_token = 128
    with pytest.raises(ValueError, match="lengths_out"):
        nat.call("kab_kv_pages_evict", ctypes.byref(p), 512, 4, 8, 2, 2, 1024, 256, None)
