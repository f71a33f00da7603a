"""The paged FP8 KV cache in numpy: the append and the eviction bit for bit, the attention in
64 bits. Pages are uint8 e4m3 codes ``[num_pages, kv_heads, page_tokens, head_dim]`` with fp32
scales ``[num_pages, kv_heads]``; the append and the eviction change the arrays they are given."""

from __future__ import annotations

import numpy as np

from .formats import e4m3_from_f32, e4m3_to_f32


def page_scale(amax: float) -> np.float32:
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    if amax == 0:
        return np.float32(2.0 ** -126)
    m, e = np.frexp(np.float64(amax))  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return np.float32(2.0 ** min(max(int(e) - 9 + (m > 0.875), -126), 120))


def _amax(x: np.ndarray) -> float:
    x = np.abs(x[np.isfinite(x)])
    return float(x.max()) if x.size else 0.0


def _codes(x: np.ndarray) -> np.ndarray:
    """e4m3 codes of fp32 values: saturating, NaN as 0x7F."""
    out = e4m3_from_f32(np.clip(x, -448, 448).astype(np.float32))
    return np.where(np.isnan(x), np.uint8(0x7F), out)


def append(k, v, k_pages, k_scale, v_pages, v_scale, table, lengths, counts=None, mass=None) -> np.ndarray:
    page = k_pages.shape[2]
    batch, heads, new, _ = k.shape
    counts = [new] * batch if counts is None else counts
    for b in range(batch):
        lo, end = int(lengths[b]), int(lengths[b]) + int(counts[b])
        while lo < end:
            hi = min(end, (lo // page + 1) * page)
            p, a = int(table[b][lo // page]), lo % page
            for codes, scale, x in ((k_pages, k_scale, k), (v_pages, v_scale, v)):
                for h in range(heads):
                    fresh = x[b, h, lo - lengths[b]:hi - lengths[b]].astype(np.float32)
                    s = page_scale(_amax(fresh))
                    if a:
                        old = scale[p, h]
                        s = max(s, old)
                        if s != old:
                            codes[p, h, :a] = _codes(e4m3_to_f32(codes[p, h, :a]) * old / s)
                    codes[p, h, a:a + hi - lo] = _codes(fresh / s)
                    scale[p, h] = s
            if mass is not None:
                mass[p, :, a:a + hi - lo] = 0
            lo = hi
    return np.array([int(a) + int(c) for a, c in zip(lengths, counts)], np.int32)


def values(pages, scale, table, length) -> np.ndarray:
    """The cached values of one sequence ``[kv_heads, length, head_dim]`` in float64."""
    page = pages.shape[2]
    at = np.asarray(table[:-(-length // page)], np.int64)
    x = e4m3_to_f32(pages[at]).astype(np.float64) * scale[at].astype(np.float64)[:, :, None, None]
    return x.transpose(1, 0, 2, 3).reshape(pages.shape[1], -1, pages.shape[3])[:, :length]


def attention(q, k_pages, k_scale, v_pages, v_scale, table, lengths, scale=None, causal=True):
    """``(out, received, size)``: the attention of q ``[B, Hq, Lq, D]``, each sequence's
    ``[kv_heads, length]`` received weight, and ``sum p |v|``, the size that roundings of p act on."""
    batch, hq, lq, d = q.shape
    heads = k_pages.shape[1]
    out = np.zeros(q.shape, np.float64)
    size = np.zeros(q.shape, np.float64)
    received = []
    for b in range(batch):
        n = int(lengths[b])
        k, v = values(k_pages, k_scale, table[b], n), values(v_pages, v_scale, table[b], n)
        got = np.zeros((heads, n))
        for h in range(hq):
            kv = h // (hq // heads)
            for i in range(lq):
                seen = max(0, n - lq + 1 + i) if causal else n
                if seen == 0:
                    continue
                s = k[kv, :seen] @ q[b, h, i].astype(np.float64) * (d ** -0.5 if scale is None else scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, h, i] = p @ v[kv, :seen]
                size[b, h, i] = p @ np.abs(v[kv, :seen])
                got[kv, :seen] += p
        received.append(got)
    return out, received, size


def keep(mass: np.ndarray, length: int, budget: int, recent: int, sinks: int) -> np.ndarray:
    """The kept token numbers of one (sequence, head), in order."""
    if length <= budget:
        return np.arange(length)
    middle = np.arange(sinks, length - recent)
    m = mass[middle].astype(np.float64)
    m = np.where(np.isnan(m), np.inf, m)  # NaN, then +inf, share the top: told apart by the first key
    order = np.lexsort((middle, -m, ~np.isnan(mass[middle])))
    chosen = middle[np.sort(order[:budget - recent - sinks])]
    return np.concatenate([np.arange(sinks), chosen, np.arange(length - recent, length)])


def evict(k_pages, k_scale, v_pages, v_scale, mass, table, lengths, to, budget, recent=0, sinks=0):
    page, heads = k_pages.shape[2], k_pages.shape[1]
    kept = np.full((len(lengths), heads, budget), -1, np.int32)
    before = [a.copy() for a in (k_pages, k_scale, v_pages, v_scale, mass)]
    for b, n in enumerate(int(x) for x in lengths):
        pages = np.asarray(table[b][:-(-n // page)], np.int64)
        for h in range(heads):
            held = before[4][pages, h].reshape(-1)[:n]
            index = keep(held, n, budget, recent, sinks)
            kept[b, h, :index.size] = index
            for j in range(-(-index.size // page)):
                part = index[j * page:(j + 1) * page]
                src, slot, dst = pages[part // page], part % page, int(to[b][j])
                mass[dst, h, :part.size] = before[4][src, h, slot]
                for codes, scale, oc, os in ((k_pages, k_scale, before[0], before[1]),
                                             (v_pages, v_scale, before[2], before[3])):
                    x = e4m3_to_f32(oc[src, h, slot]) * os[src, h][:, None]
                    s = page_scale(_amax(x))
                    codes[dst, h, :part.size] = _codes(x / s)
                    scale[dst, h] = s
    return kept, np.minimum(np.asarray(lengths), budget).astype(np.int32)
