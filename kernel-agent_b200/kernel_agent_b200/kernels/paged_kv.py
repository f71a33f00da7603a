"""A paged FP8 KV cache with one scale per (page, KV head): append, attention, eviction.

Where :mod:`kernel_agent_b200.kernels.kv_quant` holds one contiguous cache per batch with a scale
per (token, head), this cache is a pool of pages that sequences of any lengths share through a
page table, and the scales shrink to one per page and head. A page's scale is a power of two, so
a page that grows past it, or tokens that move to another page, keep their values (but for codes
that become subnormal).

* :func:`append_kv_pages`: quantise new tokens into their slots (prompts and single tokens).
* :func:`paged_kv_attention`: attention of the newest tokens over the pages; optionally adds the
  weight that every cached token received to its ``mass``.
* :func:`evict_kv_pages`: keep the first, the newest and the heaviest tokens, in other pages.
* :class:`PagedFp8KVCache`: the pool, its page table and its free pages.

K and V pages are ``[num_pages, kv_heads, page_tokens, head_dim]`` e4m3 (views with other strides
are fine, the last one 1), their scales ``[num_pages, kv_heads]`` fp32, ``mass [num_pages,
kv_heads, page_tokens]`` fp32; ``page_table [batch, max_pages]`` and ``lengths [batch]`` int32, on
the device. The kernels check page numbers and lengths themselves: a bad one is skipped and raises
bit 2 of :func:`kernel_agent_b200._native.device_status`.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native as nat
from ._launch import call, device_of, keep, stream_of, to_device, workspace

_E4M3 = torch.float8_e4m3fn
PAGE_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_TEMPLATES: dict[tuple, tuple] = {}


def _strides(t: torch.Tensor) -> list[int]:
    """The strides of the first three dimensions, 0 along those of size 1, whose strides mean nothing."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape)]


def _pool_fields(p, k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths) -> None:
    """Checks the cache's tensors and fills everything of ``p`` but the pointers."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError(f"pages must be [num_pages, kv_heads, page_tokens, head_dim]; got K {tuple(k_pages.shape)}, "
                         f"V {tuple(v_pages.shape)}")
    if k_pages.dtype != _E4M3 or v_pages.dtype != _E4M3:
        raise ValueError("the pages must be float8_e4m3fn")
    pages, heads, page, dim = k_pages.shape
    if heads < 1:
        raise ValueError("the pages need at least one KV head")
    if page not in PAGE_TOKENS:
        raise ValueError(f"page_tokens {page}: one of {', '.join(map(str, PAGE_TOKENS))}")
    if dim not in HEAD_DIMS:
        raise ValueError(f"head_dim {dim}: the paged cache takes 64 or 128")
    for name, t, shape in (("k_scale", k_scale, (pages, heads)), ("v_scale", v_scale, (pages, heads)),
                           ("mass", mass, (pages, heads, page))):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != shape):
            raise ValueError(f"{name} must be float32 {list(shape)}; got {t.dtype} {tuple(t.shape)}")
    if mass is not None and mass.stride(2) != 1:
        raise ValueError("mass needs a unit last stride")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("the pages need a unit last stride")
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError(f"page_table must be int32 [batch, max_pages]; got {page_table.dtype} "
                         f"{tuple(page_table.shape)}")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table needs a unit last stride")
    batch = page_table.shape[0]
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be int32 [{batch}], contiguous; got {lengths.dtype} {tuple(lengths.shape)}")
    p.k_stride_page, p.k_stride_head, p.k_stride_token = _strides(k_pages)
    p.v_stride_page, p.v_stride_head, p.v_stride_token = _strides(v_pages)
    p.ks_stride_page, p.ks_stride_head = k_scale.stride()
    p.vs_stride_page, p.vs_stride_head = v_scale.stride()
    if mass is not None:
        p.mass_stride_page, p.mass_stride_head = mass.stride()[:2]
    p.num_pages, p.heads_kv, p.page_tokens, p.head_dim = pages, heads, page, dim
    p.table_stride, p.max_pages, p.batch = page_table.stride(0), page_table.shape[1], batch


def _layout(k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths) -> tuple:
    """Everything of a cache's tensors that the checks and the parameters go by, but the pointers."""
    return (k_pages.shape, k_pages.stride(), k_pages.dtype, k_scale.shape, k_scale.stride(), k_scale.dtype,
            v_pages.shape, v_pages.stride(), v_pages.dtype, v_scale.shape, v_scale.stride(), v_scale.dtype,
            page_table.shape, page_table.stride(), page_table.dtype, lengths.shape, lengths.stride(), lengths.dtype,
            None if mass is None else (mass.shape, mass.stride(), mass.dtype))


def _pointers(p, k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths) -> None:
    p.k_pages, p.k_scale = k_pages.data_ptr(), k_scale.data_ptr()
    p.v_pages, p.v_scale = v_pages.data_ptr(), v_scale.data_ptr()
    if mass is not None:
        p.mass = mass.data_ptr()
    p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()


def _pool(cache: tuple) -> "nat.KabKvPages":
    """The parameters of a cache; the checks run once per layout."""
    key = _layout(*cache)
    made = _TEMPLATES.get(key)
    if made is None:
        p = nat.KabKvPages()
        _pool_fields(p, *cache)
        made = keep(_TEMPLATES, key, (bytes(p),))
    p = nat.KabKvPages.from_buffer_copy(made[0])
    _pointers(p, *cache)
    return p


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, list[int]]:
    """Rows that the kernels can load 16 bytes at a time, and their strides."""
    strides = _strides(t)
    if t.stride(3) != 1 or any(s % 8 for s in strides) or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)  # contiguous() would leave a tensor off 16 bytes there
        strides = _strides(t)
    return t, strides


def append_kv_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, k_scale: torch.Tensor,
                    v_pages: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    counts: torch.Tensor | None = None, mass: torch.Tensor | None = None,
                    out_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Write the first ``counts[b]`` (default: all) tokens of ``k``, ``v [batch, kv_heads, new,
    head_dim]`` (bf16, fp16 or fp32) after the ``lengths[b]`` cached tokens of each sequence, into
    the pages that ``page_table`` gives them; returns the new lengths (``out_lengths`` if given,
    which may be ``lengths`` itself).

    A page's scale is the smallest power of two ``s >= 2**-126`` with ``|x| <= 448 s`` for every
    finite value appended to it; codes are ``e4m3(x / s)``, to nearest even. Appending to a page
    that would need a larger scale rewrites the page's codes as ``e4m3(code * old / s)``. An
    infinity becomes the largest code of its sign, NaN stays NaN. ``mass`` of the new slots
    becomes 0. A page that receives tokens must be one sequence's own."""
    device = device_of(k, v, k_pages, k_scale, v_pages, v_scale, page_table, lengths, counts, mass, out_lengths)
    p = _pool((k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths))
    if k.dim() != 4 or v.shape != k.shape or k.shape[0] != p.batch or k.shape[1] != p.heads_kv \
            or k.shape[3] != p.head_dim:
        raise ValueError(f"expected k and v [{p.batch}, {p.heads_kv}, new, {p.head_dim}]; got {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if k.dtype != v.dtype or k.dtype not in nat.DTYPES:
        raise ValueError(f"k and v must both be float32, bfloat16 or float16; got {k.dtype}, {v.dtype}")
    for name, t in (("counts", counts), ("out_lengths", out_lengths)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (p.batch,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be int32 [{p.batch}], contiguous; got {t.dtype} {tuple(t.shape)}")
    (k, k_strides), (v, v_strides) = _rows16(k), _rows16(v)
    out = torch.empty_like(lengths) if out_lengths is None else out_lengths
    call("kab_kv_pages_append", device, ctypes.byref(p), k.data_ptr(), v.data_ptr(), nat.DTYPES[k.dtype],
         *k_strides, *v_strides, k.shape[2], nat.ptr(counts), out.data_ptr(), stream_of(device))
    return out


def paged_kv_attention(q: torch.Tensor, k_pages: torch.Tensor, k_scale: torch.Tensor, v_pages: torch.Tensor,
                       v_scale: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                       scale: float | None = None, causal: bool = True, mass: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(Q Kᵀ · scale) V over the pages, in ``q``'s dtype: ``q [B, Hq, D]`` (one query token
    per sequence) or ``[B, Hq, Lq, D]`` (bf16, fp16 or fp32; Hq a multiple of the cache's KV
    heads), ``scale`` default ``D ** -0.5``.

    With ``causal`` the queries are the newest ``Lq`` cached tokens: query i sees the first
    ``lengths[b] - Lq + 1 + i`` tokens; without it every query sees every token. A query that sees
    nothing gives zeros. With ``mass``, the weight of every cached token, summed over the query
    heads of its KV head and the query tokens, is added to its entry; pages of a common prefix may stand
    in several rows of the table and receive from each (in no fixed order). Made for the few rows (query
    heads per KV head x query tokens) of a decode step: each 16 rows (8 or 4 where there are no more)
    read the cache once. A prompt is right too, and slow (4 x 2048 tokens, 32 query heads: 19 ms).
    ``mass`` takes scratch memory of four bytes per query row and token that the page table has room
    for, at most 256 MB: where that is more, sequences or query tokens go in parts.
    Results do not depend on the other sequences' lengths but in the last bits (the cache is cut into
    equal parts for the GPU, whose softmax sums are merged), and are the same for the same
    inputs."""
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, Hq, D] or [B, Hq, Lq, D]; got {tuple(q.shape)}")
    device = device_of(q, k_pages, k_scale, v_pages, v_scale, page_table, lengths, mass, out)
    if q.dtype not in nat.DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype} (float32, bfloat16 or float16)")
    q4 = q if q.dim() == 4 else q.unsqueeze(2)
    if q4.stride(3) != 1:
        q4 = q4.contiguous()
    if scale is not None:
        scale = float(scale)  # the value: a tensor would be looked up by its identity
    cache = (k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths)
    key = ("attention", q4.shape, q4.stride(), q4.dtype, device, scale, bool(causal), _layout(*cache))
    made = _TEMPLATES.get(key)
    if made is None:
        t = nat.KabKvPagesAttention()
        _pool_fields(t.cache, *cache)
        b, hq, lq, d = q4.shape
        if b != t.cache.batch or d != t.cache.head_dim or hq % t.cache.heads_kv:
            raise ValueError(f"q {tuple(q.shape)} does not fit the cache: {t.cache.batch} sequences, "
                             f"{t.cache.heads_kv} KV heads, head_dim {t.cache.head_dim}")
        t.q_dtype, t.causal, t.use_mass = nat.DTYPES[q4.dtype], int(bool(causal)), int(mass is not None)
        t.sm_scale = d ** -0.5 if scale is None else scale
        t.q_stride_b, t.q_stride_h, t.q_stride_t = q4.stride()[:3]
        t.heads_q, t.q_len = hq, lq
        _pointers(t.cache, *cache)
        nbytes = ctypes.c_size_t(0)
        call("kab_kv_pages_attention_workspace", device, ctypes.byref(t), ctypes.byref(nbytes))
        made = keep(_TEMPLATES, key, (bytes(t), int(nbytes.value)))
    template, nbytes = made
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"out must be {q.dtype} {list(q.shape)}, contiguous; got {out.dtype} {tuple(out.shape)}")
    p = nat.KabKvPagesAttention.from_buffer_copy(template)
    _pointers(p.cache, *cache)
    p.q, p.out = q4.data_ptr(), out.data_ptr()
    stream = stream_of(device)
    ws = workspace(device, nbytes) if nbytes else None
    call("kab_kv_pages_attention", device, ctypes.byref(p), nat.ptr(ws), nbytes, stream)
    return out


def evict_kv_pages(k_pages: torch.Tensor, k_scale: torch.Tensor, v_pages: torch.Tensor, v_scale: torch.Tensor,
                   mass: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, out_page_table: torch.Tensor,
                   *, budget: int, recent: int = 0, sinks: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Keep ``min(lengths[b], budget)`` tokens of every (sequence, KV head) and copy them, in their
    order, into the pages of ``out_page_table [batch, >= ceil(budget / page_tokens)]``: pages of the
    same pool that no sequence uses (the old ones are free afterwards). Kept are the first
    ``sinks`` tokens, the last ``recent`` and, of the others, those of the largest ``mass`` (equal
    masses: the first; NaN counts as the largest). Codes move to the smallest power-of-two scale
    that holds the page's new tokens; masses move along.

    Returns ``(kept [batch, kv_heads, budget] int32, lengths [batch] int32)``: the kept token
    numbers (-1 past the last) and the new lengths."""
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if mass is None:
        raise ValueError("an eviction needs the tokens' mass")
    device = device_of(k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths, out_page_table)
    p = _pool((k_pages, k_scale, v_pages, v_scale, mass, page_table, lengths))
    if budget < 1 or recent < 0 or sinks < 0 or sinks + recent > budget:
        raise ValueError(f"budget {budget} must be at least 1 and hold the {sinks} first and {recent} last tokens")
    need = min(-(-budget // p.page_tokens), max(p.max_pages, 1))
    if out_page_table.dtype != torch.int32 or out_page_table.dim() != 2 or out_page_table.shape[0] != p.batch \
            or out_page_table.shape[1] < need or (out_page_table.shape[1] > 1 and out_page_table.stride(1) != 1):
        raise ValueError(f"out_page_table must be int32 [{p.batch}, >= {need}] with a unit last stride; got "
                         f"{out_page_table.dtype} {tuple(out_page_table.shape)}")
    if out_page_table.data_ptr() == page_table.data_ptr() and page_table.numel():
        raise ValueError("out_page_table must name other pages than page_table")
    kept = lengths.new_empty((p.batch, p.heads_kv, budget))
    out = torch.empty_like(lengths)
    call("kab_kv_pages_evict", device, ctypes.byref(p), out_page_table.data_ptr(), out_page_table.stride(0), budget,
         recent, sinks, kept.data_ptr(), out.data_ptr(), stream_of(device))
    return kept, out


class PagedFp8KVCache:
    """A pool of FP8 pages with the page table, lengths and free pages of ``batch`` sequences.

    :meth:`append` takes pages as sequences grow, :meth:`attend` reads the cache (and, with ``mass``,
    keeps every token's received weight), :meth:`evict` cuts sequences to a budget of tokens and
    frees the pages they leave, :meth:`free` ends a sequence. Page numbers are kept on the host, so
    nothing waits for the GPU; the calls follow one another on the current stream. A step captured
    in a CUDA graph calls the functions of this module on :attr:`pool` after :meth:`reserve`; its replays
    move :attr:`lengths` alone, so :meth:`advance` has to tell the host what they appended before the next
    call of another method here."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, num_pages: int, page_tokens: int = 64,
                 max_pages: int | None = None, mass: bool = True, device: torch.device | str | None = None) -> None:
        if page_tokens not in PAGE_TOKENS:
            raise ValueError(f"page_tokens {page_tokens}: one of {', '.join(map(str, PAGE_TOKENS))}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {head_dim}: the paged cache takes 64 or 128")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dev.type != "cuda":
            raise ValueError("CUDA device required (kernel_agent_b200 runs on the GPU only)")
        shape = (num_pages, kv_heads, page_tokens, head_dim)
        self.k_pages = torch.zeros(shape, dtype=_E4M3, device=dev)
        self.v_pages = torch.zeros(shape, dtype=_E4M3, device=dev)
        self.k_scale = torch.ones(shape[:2], dtype=torch.float32, device=dev)
        self.v_scale = torch.ones(shape[:2], dtype=torch.float32, device=dev)
        self.mass = torch.zeros(shape[:3], dtype=torch.float32, device=dev) if mass else None
        self.max_pages = num_pages if max_pages is None else max_pages
        self.page_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.page_tokens = page_tokens
        #: Cached tokens of each sequence, as the host knows them.
        self.tokens = [0] * batch
        self._pages: list[list[int]] = [[] for _ in range(batch)]
        self._free = list(range(num_pages - 1, -1, -1))

    @property
    def pool(self) -> tuple[torch.Tensor, ...]:
        """``(k_pages, k_scale, v_pages, v_scale, page_table, lengths)``, as the functions take them."""
        return self.k_pages, self.k_scale, self.v_pages, self.v_scale, self.page_table, self.lengths

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _table(self) -> torch.Tensor:
        """The columns of the page table that any sequence has pages in: launches and scratch memory of the
        functions follow its width."""
        return self.page_table[:, :max(1, max(map(len, self._pages), default=1))]

    def _write_table(self, changed: list[tuple[int, int, int]]) -> None:
        """Writes the entries ``[first, last)`` of the sequences in ``changed`` (sequence, first, last)."""
        at = [(b, i) for b, first, last in changed for i in range(first, last)]
        if not at:
            return
        # -1 past a sequence's pages: a kernel that comes there skips it and reports it
        pages = [self._pages[b][i] if i < len(self._pages[b]) else -1 for b, i in at]
        sent = to_device([[b * self.max_pages + i for b, i in at], pages], torch.int64, self.page_table.device)
        self.page_table.view(-1).index_copy_(0, sent[0], sent[1].to(torch.int32))

    def _not_captured(self) -> None:
        # neither the host's counts nor the host memory of a table's copy would be there for a replay
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the cache counts tokens on the host: reserve() first and capture append_kv_pages")

    def _check_counts(self, counts: list[int]) -> None:
        if len(counts) != len(self.tokens) or min(counts, default=0) < 0:
            raise ValueError(f"counts must be {len(self.tokens)} numbers of tokens; got {counts}")

    def reserve(self, counts: list[int]) -> None:
        """Take the pages that ``counts[b]`` more tokens of each sequence than :attr:`tokens` need."""
        self._check_counts(counts)
        need = [max(0, -(-(t + c) // self.page_tokens) - len(p)) for t, c, p in zip(self.tokens, counts, self._pages)]
        if sum(need) > len(self._free):
            raise ValueError(f"paged KV cache full: {sum(need)} pages wanted, {len(self._free)} free")
        if any(len(p) + n > self.max_pages for p, n in zip(self._pages, need)):
            raise ValueError(f"a sequence would pass {self.max_pages} pages")
        if any(need):
            self._not_captured()
            held = [len(p) for p in self._pages]
            for pages, n in zip(self._pages, need):
                pages += [self._free.pop() for _ in range(n)]
            self._write_table([(b, held[b], held[b] + n) for b, n in enumerate(need)])

    def advance(self, counts: list[int]) -> None:
        """Count ``counts[b]`` tokens of each sequence that replays of a captured step have appended through
        :attr:`pool` (the device's lengths moved with them), within what :meth:`reserve` took pages for."""
        self._check_counts(counts)
        if any(t + c > len(p) * self.page_tokens for t, c, p in zip(self.tokens, counts, self._pages)):
            raise ValueError(f"counts {counts} pass the pages held: reserve() before the steps that append them")
        self.tokens = [t + c for t, c in zip(self.tokens, counts)]

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: list[int] | None = None) -> None:
        """Append ``k``, ``v [batch, kv_heads, new, head_dim]``, the first ``counts[b]`` tokens of each
        sequence (default: all), as :func:`append_kv_pages` does."""
        self._not_captured()
        if k.dim() != 4:
            raise ValueError(f"expected k and v [batch, kv_heads, new, head_dim]; got {tuple(k.shape)}")
        new = k.shape[2]
        each = [new] * len(self.tokens) if counts is None else [int(c) for c in counts]
        if any(c < 0 or c > new for c in each):
            raise ValueError(f"counts must lie in 0..{new}; got {each}")
        self.reserve(each)
        count = None if counts is None else to_device(each, torch.int32, self.lengths.device)
        append_kv_pages(k, v, *self.pool, counts=count, mass=self.mass, out_lengths=self.lengths)
        self.tokens = [t + c for t, c in zip(self.tokens, each)]

    def attend(self, q: torch.Tensor, scale: float | None = None, causal: bool = True) -> torch.Tensor:
        """:func:`paged_kv_attention` of ``q`` over the cache; adds to :attr:`mass` where there is one."""
        return paged_kv_attention(q, self.k_pages, self.k_scale, self.v_pages, self.v_scale, self._table(),
                                  self.lengths, scale=scale, causal=causal, mass=self.mass)

    def evict(self, budget: int, recent: int = 0, sinks: int = 0) -> tuple[list[int], torch.Tensor | None]:
        """Cut every sequence of more than ``budget`` tokens to ``budget``, as :func:`evict_kv_pages`
        does, and free the pages it leaves. Returns ``(sequences, kept)``: which were cut, and their
        kept token numbers ``[len(sequences), kv_heads, budget]`` (None if none were)."""
        if self.mass is None:
            raise ValueError("an eviction needs the tokens' mass: make the cache with mass=True")
        if budget < 1 or recent < 0 or sinks < 0 or sinks + recent > budget:
            raise ValueError(f"budget {budget} must be at least 1 and hold the {sinks} first and {recent} last tokens")
        over = [b for b, n in enumerate(self.tokens) if n > budget]
        if not over:
            return [], None
        self._not_captured()
        each = -(-budget // self.page_tokens)
        if each * len(over) > len(self._free):
            raise ValueError(f"paged KV cache full: an eviction moves into {each * len(over)} pages, "
                             f"{len(self._free)} free")
        taken = self._free[len(self._free) - each * len(over):]
        to = [taken[i * each:(i + 1) * each] for i in range(len(over))]
        dev = self.lengths.device
        which = to_device(over, torch.int64, dev)
        target = to_device(to, torch.int32, dev)
        kept, lengths = evict_kv_pages(self.k_pages, self.k_scale, self.v_pages, self.v_scale, self.mass,
                                       self._table()[which], self.lengths[which], target, budget=budget,
                                       recent=recent, sinks=sinks)
        self.lengths[which] = lengths
        del self._free[len(self._free) - len(taken):]
        changed = []
        for b, pages in zip(over, to):
            changed.append((b, 0, max(len(pages), len(self._pages[b]))))
            self._free += self._pages[b]
            self._pages[b], self.tokens[b] = pages, budget
        self._write_table(changed)
        return over, kept

    def free(self, sequence: int) -> None:
        """End a sequence: its pages are free, its row of the batch is empty."""
        self._not_captured()
        sequence = range(len(self.tokens))[sequence]
        held = len(self._pages[sequence])
        self._free += self._pages[sequence]
        self._pages[sequence], self.tokens[sequence] = [], 0
        self.lengths[sequence] = 0
        self._write_table([(sequence, 0, held)])
