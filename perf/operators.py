"""What one generated token costs when the weights are held in 4 bits and the key / value cache in
8 bits with a scale per page and head: the cases of the four operators of that step, their plain
forms and their values in 64 bits.

* ``linear``: ``x @ Wᵀ (+ bias)`` for a few tokens, the activations as they are and the weight in
  NVFP4 (e2m1 codes, e4m3 scales per 16) or MXFP4 (e8m0 scales per 32).
* ``append``: new keys and values into the pages of an e4m3 cache, one power-of-two scale per
  (page, KV head); a page that grows past its scale is held at the larger one.
* ``attend``: attention of the newest tokens over such a cache, and the weight that every cached
  token received added to its ``mass``.
* ``evict``: the tokens a sequence keeps (the first, the newest and those of the largest mass),
  moved into other pages.

With ``own`` false ``run`` computes an operator in its plain form (elementary torch operations in
32 bits); with ``own`` true it calls ``kernel_agent_b200.kernels``.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_E4M3 = torch.float8_e4m3fn
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_BLOCK = {"nvfp4": 16, "mxfp4": 32}


def _ops():
    """The package's modules (its folder is beside this file's)."""
    package = str(Path(__file__).resolve().parents[1] / "kernel-agent_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from kernel_agent_b200.kernels import gemv, paged_kv

    return gemv, paged_kv


# ------------------------------------------------------------------ the cases


def _linear(name, m, n, k, fmt, dtype, bias=False, blocked=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "fmt": fmt, "dtype": dtype, "bias": bias,
            "blocked": blocked}


def _append(name, batch, heads, dim, page, cached, new, dtype, ragged):
    return {"name": name, "op": "append", "batch": batch, "heads": heads, "dim": dim, "page": page,
            "cached": cached, "new": new, "dtype": dtype, "ragged": ragged}


def _attend(name, batch, heads_q, heads, dim, page, tokens, queries, dtype, ragged, mass):
    return {"name": name, "op": "attend", "batch": batch, "heads_q": heads_q, "heads": heads, "dim": dim,
            "page": page, "tokens": tokens, "queries": queries, "dtype": dtype, "ragged": ragged, "mass": mass}


def _evict(name, batch, heads, dim, page, tokens, budget, recent, sinks, ragged):
    return {"name": name, "op": "evict", "batch": batch, "heads": heads, "dim": dim, "page": page,
            "tokens": tokens, "budget": budget, "recent": recent, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # one token through the smallest configuration's weight: latency alone
        _linear("linear 1x1024x1024", 1, 1024, 1024, "nvfp4", "bf16", bias=True),
        # one token through the W4A4 configuration's weight: the weight stream alone
        _linear("linear 1x28672x8192", 1, 28672, 8192, "nvfp4", "bf16", bias=True),
        # a batch of eight through the MLP's down projection, scales in the layout the GEMMs read
        _linear("linear 8x4096x14336 mx", 8, 4096, 14336, "mxfp4", "bf16", blocked=True),
        # a speculative step through a projection whose sizes are no multiple of anything
        _linear("linear 5x1001x4080 f16", 5, 1001, 4080, "nvfp4", "f16"),
        # prompts of unequal length entering the cache
        _append("append prompts 4x2048", 4, 8, 128, 64, 0, 2048, "bf16", True),
        # one token of each of many sequences: partly filled pages, some of which grow
        _append("append 64 tokens", 64, 8, 128, 64, 1000, 1, "bf16", True),
        # a single sequence with a short cache
        _attend("attend 1x4096", 1, 32, 8, 128, 64, 4096, 1, "bf16", False, False),
        # a served batch of unequal lengths, with the weights that eviction goes by
        _attend("attend 32x8192 mass", 32, 32, 8, 128, 64, 8192, 1, "bf16", True, True),
        # a few long documents, two KV heads: the cache stream alone
        _attend("attend 4x131072", 4, 16, 2, 128, 128, 131072, 1, "bf16", False, False),
        # four drafted tokens per sequence, narrow heads, small pages, empty and one-token caches
        _attend("attend 9x4x1500 f16", 9, 12, 4, 64, 16, 1500, 4, "f16", True, True),
        # one long document cut to an eighth
        _evict("evict 1x32768", 1, 8, 128, 64, 32768, 4096, 1024, 4, False),
        # a served batch, some of it shorter than the budget
        _evict("evict 16x8192", 16, 8, 128, 64, 8192, 2048, 512, 4, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "append", "attend", "attend", "evict"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "linear":
        fmt = rng.choice(("nvfp4", "mxfp4"))
        block = _BLOCK[fmt]
        while True:
            k, n = block * _log(rng, 256 / block, 14336 / block), _log(rng, 200, 28672)
            if n * k <= 28672 * 8192 and 3072 not in (n, k):
                break
        blocked = k % 256 == 0 and rng.random() < 0.5
        case = _linear("", rng.choice((1, 1, 2, 3, 4, 7, 8, 12, 16, 19, 32)), n, k, fmt, dtype, rng.random() < 0.5,
                       blocked)
    else:
        heads, dim, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), rng.choice((16, 32, 64, 128))
        batch = _log(rng, 1, 48)
        ragged = rng.random() < 0.7
        if op == "append":
            new, cached = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 16, 4096))), _log(rng, 1, 4000)
            new, cached = new + (new == 3072), cached + (cached == 3072)
            batch = max(1, min(batch, 16384 // new))
            case = _append("", batch, heads, dim, page, cached, new, dtype, ragged)
        else:
            most = 4 * 2 * 131072 * 128 // (batch * heads * dim)
            tokens = min(_log(rng, 16, 65536), most) + rng.randint(0, 15)
            tokens += tokens == 3072
            if op == "attend":
                group, queries = rng.choice((1, 2, 4, 5, 8)), rng.choice((1, 1, 1, 2, 3, 4))
                case = _attend("", batch, heads * group, heads, dim, page, tokens, queries, dtype, ragged,
                               rng.random() < 0.5)
            else:
                budget = max(8, int(tokens * rng.uniform(0.05, 1.1)))
                budget += budget == 3072
                recent = rng.randint(0, budget // 2)
                case = _evict("", batch, heads, dim, page, tokens, budget, recent, rng.randint(0, min(4, budget - recent)),
                              ragged)
    del case["name"]
    return case


def _lengths(case):
    """Cached tokens per sequence (before an append), by the case alone."""
    b = case["batch"]
    if case["op"] == "append":
        full = case["cached"]
        return [random.Random(full * 131 + i).randint(0, full) if case["ragged"] else full for i in range(b)]
    full = case["tokens"]
    if not case["ragged"]:
        return [full] * b
    rnd = random.Random(full * 131 + b)
    spread = [rnd.randint(full // 8, full) for _ in range(b)]
    spread[0] = full
    if b >= 8:
        spread[3], spread[5] = 0, 1
    return spread


def _counts(case):
    """New tokens per sequence of an append."""
    new = case["new"]
    if not case["ragged"] or new == 1:
        return [new] * case["batch"]
    rnd = random.Random(new * 17 + case["batch"])
    return [new] + [rnd.randint(0, new) for _ in range(case["batch"] - 1)]


def work(case):
    op, d = case["op"], case.get("dim", 0)
    if op == "linear":
        m, n, k, e = case["m"], case["n"], case["k"], _BYTES[case["dtype"]]
        weight = n * k // 2 + n * (k // _BLOCK[case["fmt"]])
        return {"bytes": weight + m * k * e + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    rows = case["heads"]
    if op == "append":
        new = sum(_counts(case))
        e = _BYTES[case["dtype"]]
        # a row of K and of V in, its codes and its mass out; the pages' scales
        return {"bytes": new * rows * (2 * d * (e + 1) + 4) + 16 * rows * (new // case["page"] + case["batch"]),
                "flops": 4 * new * rows * d}
    lengths = _lengths(case)
    total = sum(lengths)
    pages = sum(-(-n // case["page"]) for n in lengths)
    if op == "attend":
        queries = case["batch"] * case["heads_q"] * case["queries"]
        return {"bytes": total * rows * (2 * d + (8 if case["mass"] else 0)) + pages * (8 * rows + 4)
                + 2 * queries * d * _BYTES[case["dtype"]],
                "flops": 4 * total * case["heads_q"] * case["queries"] * d}
    kept = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": total * rows * 4 + kept * rows * (4 * d + 8) + case["batch"] * rows * case["budget"] * 4
            + 8 * rows * 2 * (kept // case["page"]),
            "flops": total * rows}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _pow2_scale(amax):
    """The smallest power of two s with amax <= 448 s, at least 2^-126 (fp32 amax)."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875)).clamp(-126, 120))
    return torch.where(amax > 0, s, torch.full_like(amax, 2.0 ** -126))


def _weight(case, g):
    """A trained-looking weight quantised to FP4: (codes [n, k / 2], scales [n, k / block], tensor_scale)."""
    n, k, fmt = case["n"], case["k"], case["fmt"]
    block = _BLOCK[fmt]
    w = torch.randn(n, k // block, block, generator=g, device=_DEV) * 0.02
    w *= torch.exp(0.3 * torch.randn(n, 1, 1, generator=g, device=_DEV))
    amax = w.abs().amax(-1)
    if fmt == "nvfp4":
        ts = w.abs().amax() / (6 * 448.0)
        scales = (amax / 6 / ts).clamp(2.0 ** -9, 448).to(_E4M3)
        step = scales.float() * ts
    else:
        ts = torch.ones((), device=_DEV)
        exponent = torch.frexp(amax / 6)[1]
        scales = (exponent + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        step = torch.ldexp(torch.ones_like(amax), exponent)
    v = w / step[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=_DEV)
    codes = torch.bucketize(v.abs(), edges).to(torch.uint8)
    codes |= (v < 0).to(torch.uint8) * 8
    codes = codes.reshape(n, k)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales.contiguous(), ts


def _blocked_index(rows, cols):
    """Where scale [r, c] stands in the flat 128 x 4 blocked layout."""
    r = torch.arange(rows, device=_DEV)[:, None]
    c = torch.arange(cols, device=_DEV)[None, :]
    return ((r // 128) * (-(-cols // 4)) + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4


def _pages_for(lengths, page, g, spare=0):
    """A page table [batch, most] of pages in no order, and how many pages the pool has."""
    need = [-(-n // page) for n in lengths]
    width = max(1, max(need))
    order = torch.randperm(sum(need) + spare, generator=g, device=_DEV).to(torch.int32)
    has = torch.arange(width, device=_DEV)[None, :] < torch.tensor(need, device=_DEV)[:, None]
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device=_DEV)
    table[has] = order[:sum(need)]
    return table, order[sum(need):], sum(need) + spare


def _pool(pages, heads, page, dim, g, outliers):
    """Codes and scales of a pool of pages: normal values, keys with a few loud channels."""
    x = torch.randn(pages, heads, page, dim, generator=g, device=_DEV)
    if outliers:
        x[..., torch.randperm(dim, generator=g, device=_DEV)[:max(1, dim // 32)]] *= 4.0
    scale = _pow2_scale(x.abs().amax(dim=(2, 3)))
    return (x / scale[:, :, None, None]).clamp(-448, 448).to(_E4M3), scale


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "linear":
        s["codes"], scales, s["tensor_scale"] = _weight(case, g)
        if case["blocked"]:
            rows, cols = scales.shape
            flat = torch.zeros(-(-rows // 128) * 128 * (-(-cols // 4)) * 4, dtype=torch.uint8, device=_DEV)
            flat[_blocked_index(rows, cols)] = scales.view(torch.uint8)
            scales = flat.view(scales.dtype)
        s["scales"] = scales
        t = _TYPES[case["dtype"]]
        x = torch.randn(case["m"], case["k"], generator=g, device=_DEV)
        x[:, torch.randperm(case["k"], generator=g, device=_DEV)[:max(1, case["k"] // 500)]] *= 20.0
        s["x"] = x.to(t)
        s["bias_"] = (torch.randn(case["n"], generator=g, device=_DEV) * 0.1).to(t) if case["bias"] else None
        return s
    heads, dim, page, batch = case["heads"], case["dim"], case["page"], case["batch"]
    lengths = _lengths(case)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=_DEV)
    if case["op"] == "append":
        counts = _counts(case)
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=_DEV)
        s["table"], _, pages = _pages_for([a + b for a, b in zip(lengths, counts)], page, g)
    elif case["op"] == "evict":
        spare = batch * -(-case["budget"] // page)
        s["table"], free, pages = _pages_for(lengths, page, g, spare)
        s["to"] = free.reshape(batch, -1).contiguous()
    else:
        s["table"], _, pages = _pages_for(lengths, page, g, 1)
    s["k_pages"], s["k_scale"] = _pool(pages, heads, page, dim, g, True)
    s["v_pages"], s["v_scale"] = _pool(pages, heads, page, dim, g, False)
    # weights received so far: a few tokens drew most of them, many nothing yet
    mass = torch.exp(2.0 * torch.randn(pages, heads, page, generator=g, device=_DEV) - 3.0)
    mass[torch.rand(mass.shape, generator=g, device=_DEV) < 0.2] = 0.0
    s["mass_"] = mass
    t = _TYPES[case.get("dtype", "bf16")]
    if case["op"] == "append":
        shape = (batch, heads, case["new"], dim)
        loud = torch.exp(0.5 * torch.randn(batch, heads, case["new"], 1, generator=g, device=_DEV))
        s["k"] = (torch.randn(shape, generator=g, device=_DEV) * 2.0 * loud).to(t)
        s["v"] = (torch.randn(shape, generator=g, device=_DEV) * loud).to(t)
    elif case["op"] == "attend":
        s["q"] = torch.randn(batch, case["heads_q"], case["queries"], dim, generator=g, device=_DEV).to(t)
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["op"]
    if own:
        gemv, paged = _ops()
        if op == "linear":
            return gemv.fp4_w4a16_linear(state["x"], state["codes"], state["scales"], state["tensor_scale"],
                                         state["bias_"], fmt=state["fmt"])
        cache = (state["k_pages"], state["k_scale"], state["v_pages"], state["v_scale"])
        if op == "append":
            lengths = paged.append_kv_pages(state["k"], state["v"], *cache, state["table"], state["lengths"],
                                            counts=state["counts"], mass=state["mass_"])
            return (*cache, state["mass_"], lengths)
        if op == "attend":
            mass = state["mass_"] if state["mass"] else None
            out = paged.paged_kv_attention(state["q"], *cache, state["table"], state["lengths"], mass=mass)
            return (out,) if mass is None else (out, mass)
        kept, lengths = paged.evict_kv_pages(*cache, state["mass_"], state["table"], state["lengths"], state["to"],
                                             budget=state["budget"], recent=state["recent"], sinks=state["sinks"])
        return (*cache, state["mass_"], kept, lengths)
    return {"linear": _run_linear, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[op](state)


def _run_linear(s):
    n, k, block = s["n"], s["k"], _BLOCK[s["fmt"]]
    scales = s["scales"].float()
    if s["blocked"]:
        scales = scales[_blocked_index(n, k // block)]
    codes = s["codes"]
    nibbles = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(n, k).long()
    values = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)[nibbles]
    w = (values.reshape(n, -1, block) * scales[..., None]).reshape(n, k)
    y = (s["x"].float() @ w.T) * s["tensor_scale"]
    if s["bias_"] is not None:
        y = y + s["bias_"].float()
    return y.to(s["x"].dtype)


def _run_append(s):
    page, lengths, counts = s["page"], s["lengths"].long(), s["counts"].long()
    batch, heads, new, dim = s["k"].shape
    first = lengths // page
    touched = -(-(new + page - 1) // page)  # pages that an append of `new` tokens can reach
    slot = (first[:, None] + torch.arange(touched, device=_DEV)[None, :])  # [batch, touched] logical pages
    at = slot[..., None] * page + torch.arange(page, device=_DEV)  # [batch, touched, page] token numbers
    old = at < lengths[:, None, None]
    fresh = (at >= lengths[:, None, None]) & (at < (lengths + counts)[:, None, None])
    write = fresh.any(-1)  # pages that get a token
    pages = torch.gather(s["table"].long(), 1, slot.clamp(max=s["table"].shape[1] - 1))
    token = (at - lengths[:, None, None]).clamp(0, max(new - 1, 0))
    rows = torch.arange(batch, device=_DEV)[:, None, None]
    for codes, scale, x in ((s["k_pages"], s["k_scale"], s["k"]), (s["v_pages"], s["v_scale"], s["v"])):
        value = x.float().permute(0, 2, 1, 3)[rows, token]  # [batch, touched, page, heads, dim]
        value = value.permute(0, 1, 3, 2, 4)
        size = torch.where(fresh[:, :, None, :, None] & torch.isfinite(value), value.abs(), 0.0)
        need = _pow2_scale(size.amax(dim=(3, 4)))
        before = torch.where(old.any(-1)[..., None], scale[pages], 0.0)
        now = torch.maximum(before, need)  # [batch, touched, heads]
        held = codes[pages].float() * before[..., None, None]
        value = torch.where(fresh[:, :, None, :, None], value, held) / now[..., None, None]
        value = value.clamp(-448, 448).to(_E4M3)
        keep = (old | fresh)[:, :, None, :, None] & write[:, :, None, None, None]
        value = torch.where(keep, value.view(torch.uint8), codes[pages].view(torch.uint8))
        codes.view(torch.uint8)[pages[write]] = value[write]
        scale[pages[write]] = now[write]
    mass = s["mass_"][pages]
    s["mass_"][pages[write]] = torch.where(fresh[:, :, None, :], 0.0, mass)[write]
    return s["k_pages"], s["k_scale"], s["v_pages"], s["v_scale"], s["mass_"], (lengths + counts).to(torch.int32)


def _run_attend(s):
    page, table, lengths = s["page"], s["table"].long(), s["lengths"].long()
    q = s["q"].float()
    batch, heads_q, queries, dim = q.shape
    heads = s["k_pages"].shape[1]
    k = s["k_pages"][table].float() * s["k_scale"][table][..., None, None]  # [batch, pages, heads, page, dim]
    v = s["v_pages"][table].float() * s["v_scale"][table][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(batch, heads, -1, dim)
    v = v.permute(0, 2, 1, 3, 4).reshape(batch, heads, -1, dim)
    q = q.reshape(batch, heads, -1, dim)  # the rows of a KV head: its query heads x the query tokens
    at = torch.arange(k.shape[2], device=_DEV)
    seen = lengths[:, None] - queries + 1 + torch.arange(queries, device=_DEV)  # tokens that each query sees
    visible = (at < seen[..., None]).repeat(1, heads_q // heads, 1)[:, None]  # [batch, 1, rows, tokens]
    score = (q @ k.transpose(2, 3)) * dim ** -0.5
    top = score.masked_fill(~visible, -math.inf).amax(-1, keepdim=True)
    p = torch.where(visible, torch.exp(score - top), 0.0)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    valid = at < lengths[:, None]
    out = (p @ torch.where(valid[:, None, :, None], v, 0.0)).reshape(batch, heads_q, queries, dim).to(s["q"].dtype)
    if not s["mass"]:
        return (out,)
    received = p.sum(2).reshape(batch, heads, -1, page).transpose(1, 2)  # [batch, pages, heads, page]
    used = torch.arange(table.shape[1], device=_DEV) * page < lengths[:, None]
    valid = valid.reshape(batch, -1, 1, page)[used]
    pages = table[used]
    s["mass_"][pages] = s["mass_"][pages] + torch.where(valid, received[used], 0.0)
    return out, s["mass_"]


def _keep_order(mass, at, length, budget, recent, sinks):
    """Which tokens stay: [.., budget] token numbers in order, -1 past the last."""
    keep = torch.minimum(length, torch.full_like(length, budget))
    forced = (at < sinks) | (at >= length - recent)
    key = torch.where(forced, math.inf, mass)
    key = torch.where(at < length, key, -math.inf)
    ranked = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    if ranked.shape[-1] < budget:
        ranked = torch.nn.functional.pad(ranked, (0, budget - ranked.shape[-1]), value=at.numel())
    place = torch.arange(budget, device=mass.device)
    ranked = torch.where(place < keep, ranked, 1 << 40).sort(-1).values
    return torch.where(place < keep, ranked, -1)


def _run_evict(s):
    page, table, to, budget = s["page"], s["table"].long(), s["to"].long(), s["budget"]
    lengths = s["lengths"].long()
    batch, heads = table.shape[0], s["k_pages"].shape[1]
    mass = s["mass_"][table].permute(0, 2, 1, 3).reshape(batch, heads, -1)
    at = torch.arange(mass.shape[-1], device=_DEV)
    kept = _keep_order(mass, at, lengths[:, None, None], budget, s["recent"], s["sinks"])  # [batch, heads, budget]
    width = to.shape[1] * page
    source = torch.nn.functional.pad(kept, (0, width - budget), value=-1)
    there = (source >= 0).reshape(batch, heads, -1, page).transpose(1, 2)  # [batch, pages, heads, page]
    source = source.clamp(min=0)
    rows = torch.arange(batch, device=_DEV)[:, None, None]
    column = torch.arange(heads, device=_DEV)[None, :, None]
    from_page, from_slot = table[rows, source // page], source % page
    write = there.any(-1).any(-1)
    for codes, scale in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
        value = codes.view(torch.uint8)[from_page, column, from_slot].view(_E4M3).float()
        value = value * scale[from_page, column][..., None]  # [batch, heads, width, dim]
        value = value.reshape(batch, heads, -1, page, value.shape[-1]).transpose(1, 2)
        size = torch.where(there[..., None] & torch.isfinite(value), value.abs(), 0.0)
        now = _pow2_scale(size.amax(dim=(3, 4)))
        value = (value / now[..., None, None]).clamp(-448, 448).to(_E4M3).view(torch.uint8)
        value = torch.where(there[..., None], value, codes[to].view(torch.uint8))
        codes.view(torch.uint8)[to[write]] = value[write]
        scale[to[write]] = now[write]
    moved = s["mass_"][from_page, column, from_slot].reshape(batch, heads, -1, page).transpose(1, 2)
    s["mass_"][to[write]] = torch.where(there, moved, s["mass_"][to])[write]
    return (s["k_pages"], s["k_scale"], s["v_pages"], s["v_scale"], s["mass_"], kept.to(torch.int32),
            lengths.clamp(max=budget).to(torch.int32))


# ------------------------------------------------------------------ the values in 64 bits


def _to_e4m3(x):
    """float64 values rounded to the nearest e4m3 value, ties to even, at most 448."""
    size = x.abs().clamp(max=448.0)
    exponent = torch.floor(torch.log2(size.clamp(min=2.0 ** -6))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return torch.sign(x) * (torch.round(size / step) * step)


def _scale_of(biggest):
    """The page scale of a largest magnitude (a float)."""
    if biggest == 0:
        return 2.0 ** -126
    e = math.ceil(math.log2(biggest / 448.0))
    while biggest > 448.0 * 2.0 ** e:
        e += 1
    while biggest <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** min(max(e, -126), 120)


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _exact_linear(s):
    n, k, block = s["n"], s["k"], _BLOCK[s["fmt"]]
    level = torch.tensor(_E2M1, dtype=torch.float64, device=_DEV)
    scales = s["scales"].double()
    out = torch.empty(s["m"], n, dtype=torch.float64, device=_DEV)
    x = s["x"].double()
    for lo in range(0, n, 2048):  # a panel of the weight's rows at a time
        c = s["codes"][lo:lo + 2048]
        w = torch.empty(c.shape[0], k, dtype=torch.float64, device=_DEV)
        for half, nibble in ((0, c & 15), (1, c >> 4)):
            w[:, half::2] = level[(nibble & 7).long()] * (1.0 - 2.0 * (nibble >> 3).double())
        if s["blocked"]:
            r = torch.arange(lo, lo + c.shape[0], device=_DEV)[:, None]
            j = torch.arange(k // block, device=_DEV)[None, :]
            sc = scales[(r // 128 * ((k // block + 3) // 4) + j // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + j % 4]
        else:
            sc = scales[lo:lo + 2048]
        out[:, lo:lo + 2048] = x @ (w * sc.repeat_interleave(block, 1)).T
    out = out * s["tensor_scale"].double()
    return out if s["bias_"] is None else out + s["bias_"].double()


def _exact_append(s):
    page = s["page"]
    start, count, table = s["lengths"].tolist(), s["counts"].tolist(), s["table"].tolist()
    answers = []
    for codes, scale, x in ((s["k_pages"], s["k_scale"], s["k"]), (s["v_pages"], s["v_scale"], s["v"])):
        codes, scale, x = codes.double(), scale.double(), x.double()
        for b in range(len(start)):
            lo, end = start[b], start[b] + count[b]
            while lo < end:
                hi = min(end, (lo // page + 1) * page)
                p, a = table[b][lo // page], lo % page
                new = x[b, :, lo - start[b]:hi - start[b]]  # [heads, tokens, dim]
                s_new = torch.tensor([_scale_of(v) for v in new.abs().amax(dim=(1, 2)).tolist()], device=_DEV).double()
                if a:
                    s_new = torch.maximum(s_new, scale[p])
                    codes[p, :, :a] = _to_e4m3(codes[p, :, :a] * (scale[p] / s_new)[:, None, None])
                codes[p, :, a:a + hi - lo] = _to_e4m3(new / s_new[:, None, None])
                scale[p] = s_new
                lo = hi
        answers += [codes, scale]
    mass = s["mass_"].double()
    for b in range(len(start)):
        for p in range(start[b] // page, -(-(start[b] + count[b]) // page)):
            lo, hi = max(start[b] - p * page, 0), min(start[b] + count[b] - p * page, page)
            mass[table[b][p], :, lo:hi] = 0.0
    return (*answers, mass, torch.tensor([a + b for a, b in zip(start, count)], dtype=torch.int32, device=_DEV))


def _exact_attend(s):
    page, dim, heads = s["page"], s["dim"], s["heads"]
    group, queries = s["heads_q"] // heads, s["queries"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    mass = s["mass_"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        for h in range(heads):
            if n == 0:
                continue
            k = (s["k_pages"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            v = (s["v_pages"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            received = torch.zeros(pages.numel() * page, dtype=torch.float64, device=_DEV)
            for i in range(queries):
                seen = n - queries + 1 + i
                if seen <= 0:
                    continue
                score = s["q"][b, h * group:(h + 1) * group, i].double() @ k[:seen].T / math.sqrt(dim)
                p = torch.softmax(score, -1)
                out[b, h * group:(h + 1) * group, i] = p @ v[:seen]
                received[:seen] += p.sum(0)
            mass[pages, h] += received.reshape(-1, page)
    return (out, mass) if s["mass"] else (out,)


def _exact_evict(s):
    page, budget, heads = s["page"], s["budget"], s["heads"]
    table, to = s["table"].long(), s["to"].long()
    lengths = s["lengths"].tolist()
    kept = torch.full((len(lengths), heads, budget), -1, dtype=torch.int64, device=_DEV)
    codes = [s["k_pages"].double(), s["v_pages"].double()]
    scale = [s["k_scale"].double(), s["v_scale"].double()]
    old_codes, old_scale, mass = [c.clone() for c in codes], [c.clone() for c in scale], s["mass_"].double()
    old_mass = mass.clone()
    for b, n in enumerate(lengths):
        stay = min(n, budget)
        if stay == 0:
            continue
        for h in range(heads):
            m = old_mass[table[b, :-(-n // page)], h].reshape(-1)[:n].clone()
            if n > budget:
                head, tail = min(s["sinks"], n), max(n - s["recent"], 0)
                m[:head] = math.inf
                m[tail:] = math.inf
                # the stay-th largest, then as many of the equal ones, from the first, as are still wanted
                edge = torch.topk(m, stay).values[-1]
                pick = m > edge
                equal = torch.nonzero(m == edge).flatten()[:stay - int(pick.sum())]
                pick[equal] = True
                index = torch.nonzero(pick).flatten()
            else:
                index = torch.arange(n, device=_DEV)
            kept[b, h, :stay] = index
            src, slot = table[b, index // page], index % page
            dst = to[b, torch.arange(stay, device=_DEV) // page]
            place = torch.arange(stay, device=_DEV) % page
            mass[dst, h, place] = old_mass[src, h, slot]
            for c, sc, oc, osc in zip(codes, scale, old_codes, old_scale):
                value = oc[src, h, slot] * osc[src, h][:, None]
                tops = torch.zeros(-(-stay // page) * page, dtype=torch.float64, device=_DEV)
                tops[:stay] = value.abs().amax(-1)
                new = torch.tensor([_scale_of(t) for t in tops.reshape(-1, page).amax(-1).tolist()],
                                   dtype=torch.float64, device=_DEV)
                sc[to[b, :new.numel()], h] = new
                c[dst, h, place] = _to_e4m3(value / new[torch.arange(stay, device=_DEV) // page][:, None])
    return (codes[0], scale[0], codes[1], scale[1], mass, kept.to(torch.int32),
            torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32, device=_DEV))
