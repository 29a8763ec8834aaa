"""What is measured of the decode-step operators: query/key norm with RoPE (and the append to the paged pool), the
page bookkeeping of a pool (fork, copy, free, compact), and sampling a token from logits.

``run`` computes them in plain torch, or through the framework's entry points where ``own`` is true; both work on what
``prepare`` made. ``exact`` is the definition in 64 bits, written separately.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@functools.lru_cache(maxsize=None)
def _framework():
    path = os.path.join(os.getcwd(), "reflex-infer_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kernels.attention
    import kernels.kv_cache
    import kernels.rope
    import kernels.softmax
    return kernels


# ---- cases ------------------------------------------------------------------------------------

def _append(name, B, new, ctx, hq, hkv, dim, block, dtype, tables, packed):
    return {"name": name, "op": "norm_append", "B": B, "new": new, "ctx": ctx, "hq": hq, "hkv": hkv, "dim": dim,
            "block": block, "dtype": dtype, "tables": tables, "packed": packed, "interleaved": False}


def _rope(name, tokens, ctx, hq, hkv, dim, dtype, tables, packed, interleaved):
    return {"name": name, "op": "norm_rope", "tokens": tokens, "ctx": ctx, "hq": hq, "hkv": hkv, "dim": dim,
            "dtype": dtype, "tables": tables, "packed": packed, "interleaved": interleaved}


def _fork(name, parents, children, ctx, layers, hkv, dim, block, pool, dtype):
    return {"name": name, "op": "fork", "parents": parents, "children": children, "ctx": ctx, "layers": layers,
            "hkv": hkv, "dim": dim, "block": block, "pool": pool, "dtype": dtype}


def _compact(name, pool, free, requests, layers, hkv, dim, block, dtype):
    return {"name": name, "op": "compact", "pool": pool, "free": free, "requests": requests, "layers": layers,
            "hkv": hkv, "dim": dim, "block": block, "dtype": dtype}


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p, mixed, peak):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "peak": peak}


def listed():
    return [
        # one decode step of 32 requests, 16 query / 2 kv heads: Q and K normed and rotated, K and V to the pool
        _append("append_decode_32", 32, 1, 4096, 16, 2, 128, 16, "bfloat16", "float32", True),
        # a ragged chunked-prefill batch, 1 to 64 new tokens each of 64 requests, 28 / 4 heads
        _append("append_chunks_64", 64, 64, 2048, 28, 4, 128, 16, "bfloat16", "same", True),
        # prefill of 8 x 2048 tokens, 32 / 8 heads
        _append("append_prefill_8x2048", 8, -2048, 0, 32, 8, 128, 16, "bfloat16", "float32", False),
        # the norm and rotation alone, interleaved pairs, an odd number of tokens, heads of 64 out of a packed projection
        _rope("rope_f16_inter_2047", 2047, 8192, 16, 16, 64, "float16", "same", True, True),
        # parallel sampling begins: 4 prompts fork into 32 continuations on a 16-head fp32 pool of one layer
        _fork("fork_4_to_32", 4, 32, 256, 1, 16, 64, 16, 1024, "float32"),
        # a beam step: 64 beams are rebuilt from their parents, 8 layers share one page table
        _fork("fork_64_to_256_layers", 64, 256, 8192, 8, 2, 128, 16, 32768, "bfloat16"),
        # a small fragmented pool is compacted
        _compact("compact_1k", 1000, 0.4, 16, 1, 2, 128, 16, "float16"),
        # a 65536-page pool with 40 % free is compacted, 28 / 4 heads
        _compact("compact_64k", 65536, 0.4, 64, 1, 4, 128, 16, "bfloat16"),
        # one user's chat: the usual settings, one row
        _sample("sample_1x32000", 1, 32000, "float32", 0.8, 50, 0.95, 0.0, False, 16.0),
        # 32 requests, odd vocabulary (rows start at any alignment), nucleus sampling
        _sample("sample_32x50257", 32, 50257, "bfloat16", 1.0, 0, 0.9, 0.0, False, 12.0),
        # a batch in which every request has its own settings, greedy rows and unfiltered ones among them
        _sample("sample_mixed_64x131072", 64, 131072, "bfloat16", 1.0, 0, 1.0, 0.0, True, 14.0),
        # a full batch with fp32 logits and all filters on
        _sample("sample_256x131072", 256, 131072, "float32", 0.7, 200, 0.95, 0.02, False, 14.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_append", "norm_rope", "fork", "compact", "sample", "sample"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    block = rng.choice([8, 16, 16, 32, 64])
    hkv = rng.choice([1, 2, 4, 8])
    tables = rng.choice(["float32", "same"])
    if kind == "norm_append":
        B = _log(rng, 1, 64)
        return _append(None, B, rng.choice([1, _log(rng, 2, 64), -_log(rng, 2, 40)]), _log(rng, 1, 2048),
                       hkv * rng.choice([1, 4, 7, 8]), hkv, dim, block, dtype, tables, rng.random() < 0.5)
    if kind == "norm_rope":
        return _rope(None, _log(rng, 1, 3000), _log(rng, 16, 65536), hkv * rng.choice([1, 4, 7]), hkv, dim, dtype,
                     tables, rng.random() < 0.5, rng.random() < 0.5)
    if kind == "fork":
        parents = _log(rng, 1, 48)
        ctx = _log(rng, 1, 4096)
        children = _log(rng, parents, 4 * parents)
        pool = parents * (ctx // block + 1) + children + _log(rng, 16, 2000)
        return _fork(None, parents, children, ctx, rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([64, 80, 128]),
                     block, pool, dtype)
    if kind == "compact":
        return _compact(None, _log(rng, 64, 20000), rng.uniform(0.05, 0.9), _log(rng, 1, 64), rng.choice([1, 2]),
                        rng.choice([1, 2, 4]), rng.choice([64, 80, 128]), rng.choice([8, 16]), dtype)
    rows = _log(rng, 1, 128)
    vocab = _log(rng, 1000, 200000)
    return _sample(None, rows, vocab, dtype, rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), rng.choice([0, 1, 20, 64, 1000]),
                   rng.choice([1.0, 0.5, 0.9, 0.99]), rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.3,
                   rng.uniform(4.0, 20.0))


# ---- inputs -----------------------------------------------------------------------------------

def _rope_tables(rows, dim, interleaved, dtype, dev):
    inv = 1.0 / (1e6 ** (torch.arange(0, dim // 2, dtype=torch.float64, device=dev) / (dim // 2)))
    ang = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * inv
    ang = ang.repeat_interleave(2, dim=1) if interleaved else torch.cat([ang, ang], dim=1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _qkv(case, n, g, dev, with_v):
    hq, hkv, dim, dtype = case["hq"], case["hkv"], case["dim"], DTYPES[case["dtype"]]
    heads = hq + hkv * (2 if with_v else 1)
    qkv = torch.randn(n, heads, dim, generator=g, device=dev)
    qkv *= torch.exp(0.5 * torch.randn(1, heads, 1, generator=g, device=dev))  # heads differ in size
    qkv = qkv.to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    if not case["packed"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return q, k, v


def _pool(blocks, case, g, dev):
    shape = (blocks, case["hkv"], case["block"], case["dim"])
    return torch.empty(shape, dtype=DTYPES[case["dtype"]], device=dev).normal_(generator=g)


def _new_tokens(case):
    """New tokens of each request: -new each, or between 1 and new, the same for every seed."""
    if case["new"] < 0:
        return torch.full((case["B"],), -case["new"])
    return torch.randint(1, case["new"] + 1, (case["B"],), generator=torch.Generator().manual_seed(case["B"]))


def _prepare_norm(case, g, dev):
    dtype = DTYPES[case["dtype"]]
    tdtype = torch.float32 if case["tables"] == "float32" else dtype
    s = {"op": case["op"], "eps": 1e-6, "interleaved": case["interleaved"]}
    cpu = torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=g, device=dev).item()))
    rows = case["ctx"]
    if case["op"] == "norm_append":
        B, block, new = case["B"], case["block"], _new_tokens(case)
        old = torch.randint(0, case["ctx"] + 1, (B,), generator=cpu)
        pages = (old + new + block - 1) // block
        first = torch.cumsum(pages, 0) - pages
        blocks = B * ((case["ctx"] + abs(case["new"]) + block - 1) // block) + 7
        perm = torch.randperm(blocks, generator=cpu)
        req = torch.repeat_interleave(torch.arange(B), new)
        positions = old[req] + torch.arange(int(new.sum())) - (torch.cumsum(new, 0) - new)[req]
        slots = perm[first[req] + positions // block] * block + positions % block
        rows, n = rows + abs(case["new"]), int(new.sum())
        s["slots"] = slots.to(dev)
        s["k_cache"], s["v_cache"] = _pool(blocks, case, g, dev), _pool(blocks, case, g, dev)
    else:
        n = case["tokens"]
        positions = torch.randint(0, rows, (n,), generator=cpu)
    s["q"], s["k"], s["v"] = _qkv(case, n, g, dev, case["op"] == "norm_append")
    s["positions"] = positions.to(torch.int32).to(dev)
    s["cos"], s["sin"] = _rope_tables(rows, case["dim"], case["interleaved"], tdtype, dev)
    s["wq"] = (1 + 0.2 * torch.randn(case["dim"], generator=g, device=dev)).to(dtype)
    s["wk"] = (1 + 0.2 * torch.randn(case["dim"], generator=g, device=dev)).to(dtype)
    return s


def _prepare_fork(case, g, dev):
    P, block, blocks = case["parents"], case["block"], case["pool"]
    lens = torch.randint(1, case["ctx"] + 1, (P,), generator=g, device=dev)
    lens[0] = case["ctx"]
    pages = (lens + block - 1) // block
    width = (case["ctx"] + block - 1) // block + 1
    perm = torch.randperm(blocks, generator=g, device=dev)
    first = torch.cumsum(pages, 0) - pages
    cols = torch.arange(width, device=dev)
    at = (first[:, None] + cols).clamp_(max=blocks - 1)
    table = torch.where(cols < pages[:, None], perm[at], -1)
    counts = torch.zeros(blocks, dtype=torch.int32, device=dev)
    used = torch.arange(blocks, device=dev) < pages.sum()
    counts[perm] = used.to(torch.int32)
    parents = torch.randint(0, P, (case["children"],), generator=g, device=dev, dtype=torch.int32)
    return {"op": "fork", "table": table, "lens": lens.to(torch.int32), "counts": counts, "parents": parents,
            "rows": torch.arange(P, device=dev, dtype=torch.int32), "block": block,
            "k": [_pool(blocks, case, g, dev) for _ in range(case["layers"])],
            "v": [_pool(blocks, case, g, dev) for _ in range(case["layers"])]}


def _prepare_compact(case, g, dev):
    blocks, R = case["pool"], case["requests"]
    live = torch.rand(blocks, generator=g, device=dev) >= case["free"]
    order = torch.rand(blocks, generator=g, device=dev).masked_fill_(~live, 2.0).argsort()
    n_live = live.sum()
    width = (blocks + R - 1) // R
    at = torch.arange(R * width, device=dev)
    table = torch.where(at < n_live, order[at.clamp(max=blocks - 1)], -1).view(width, R).t().contiguous()
    counts = live.to(torch.int32) * torch.randint(1, 3, (blocks,), generator=g, device=dev, dtype=torch.int32)
    return {"op": "compact", "table": table, "counts": counts,
            "k": [_pool(blocks, case, g, dev) for _ in range(case["layers"])],
            "v": [_pool(blocks, case, g, dev) for _ in range(case["layers"])]}


def _prepare_sample(case, g, dev):
    B, V = case["rows"], case["vocab"]
    # a wide floor of unlikely tokens and a few dozen likely ones, whose height differs from row to row
    logits = 2.0 * torch.randn(B, V, generator=g, device=dev)
    height = case["peak"] * (0.4 + 0.8 * torch.rand(B, 1, generator=g, device=dev))
    likely = torch.randint(0, V, (B, 48), generator=g, device=dev)
    fall = 0.35 * torch.arange(48, device=dev)
    logits.scatter_(1, likely, height - fall * torch.rand(B, 1, generator=g, device=dev))
    s = {"op": "sample", "logits": logits.to(DTYPES[case["dtype"]]),
         "u": torch.rand(B, generator=g, device=dev),
         "temperature": case["temperature"], "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
    if case["mixed"]:
        pick = lambda *v: torch.tensor(v, device=dev)[torch.randint(0, len(v), (B,), generator=g, device=dev)]  # noqa: E731
        s["temperature"] = pick(0.0, 0.6, 0.8, 1.0, 1.3)
        s["top_k"] = pick(0, 0, 1, 40, 500).to(torch.int32)
        s["top_p"] = pick(1.0, 1.0, 0.5, 0.9, 0.97)
        s["min_p"] = pick(0.0, 0.0, 0.02, 0.1)
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] in ("norm_append", "norm_rope"):
        return _prepare_norm(case, g, dev)
    return {"fork": _prepare_fork, "compact": _prepare_compact, "sample": _prepare_sample}[case["op"]](case, g, dev)


# ---- the plain forms ----------------------------------------------------------------------------

def _plain_norm_rope(x, w, cos, sin, eps, interleaved):
    n = x.float()
    n = n * torch.rsqrt((n * n).mean(-1, keepdim=True) + eps) * w.float()
    c, s = cos.float()[:, None], sin.float()[:, None]
    half = x.shape[-1] // 2
    if interleaved:
        turned = torch.stack([-n[..., 1::2], n[..., ::2]], dim=-1).flatten(-2)
    else:
        turned = torch.cat([-n[..., half:], n[..., :half]], dim=-1)
    return (n * c + turned * s).to(x.dtype)


def _plain_copy(caches, src, dst, rows=None):
    for cache in caches:
        moved = cache[src]
        if rows is not None:
            kept = torch.arange(cache.shape[2], device=src.device)[None, None, :, None] < rows[:, None, None, None]
            moved = torch.where(kept, moved, cache[dst])
        cache[dst] = moved


def _plain_fork(table, lens, parents, counts, block):
    p = parents.long()
    length = lens[p].long()
    full, rest = length // block, length % block
    rows = table[p]
    shared = torch.arange(table.shape[1], device=p.device) < full[:, None]
    child = torch.where(shared, rows, -1)
    needs = rest > 0
    free = (counts != 0).to(torch.int8).sort(stable=True).indices  # free pages first, ascending
    fresh = free[(torch.cumsum(needs, 0) - 1).clamp_(min=0)]
    counts.index_add_(0, child[shared], torch.ones(1, dtype=counts.dtype, device=p.device).expand(int(shared.sum())))
    src = rows.gather(1, full[:, None])[:, 0][needs]
    dst = fresh[needs]
    counts[dst] = 1
    child[needs, full[needs]] = dst
    return child, src, dst, rest[needs]


def _plain_free(table, rows, counts):
    entries = table[rows.long()]
    entries = entries[entries >= 0]
    counts.index_add_(0, entries, -torch.ones(1, dtype=counts.dtype, device=rows.device).expand(entries.shape[0]))
    table[rows.long()] = -1


def _plain_compact(table, counts):
    blocks = counts.shape[0]
    live = counts > 0
    n_live = live.sum()
    index = torch.arange(blocks, device=counts.device)
    src = (live & (index >= n_live)).nonzero()[:, 0].flip(0)
    dst = (~live & (index < n_live)).nonzero()[:, 0]
    page_map = torch.where(live, index, -1)
    page_map[src] = dst
    counts[dst] = counts[src]
    counts[src] = 0
    table.copy_(torch.where(table >= 0, page_map[table.clamp(min=0)], table))
    return page_map, src, dst


def _column(value, B, dev, dtype):
    return value.to(dtype)[:, None] if torch.is_tensor(value) else torch.full((B, 1), value, dtype=dtype, device=dev)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    # 64 bits: a token is decided by on which side of a border a running sum lies
    B, V = logits.shape
    dev = logits.device
    index = torch.arange(V, device=dev)
    values = logits.float() + 0.0
    values = torch.where(values.isnan(), -math.inf, values)
    top = values.amax(1, keepdim=True)
    greedy = torch.where(values == top, index, V).amin(1)
    # a setting is a 32-bit number, whether it comes as a tensor or as a Python number
    T = _column(temperature, B, dev, torch.float32).double()
    p = _column(top_p, B, dev, torch.float32).double()
    least = _column(min_p, B, dev, torch.float32).double().clamp(max=1.0)
    k = _column(top_k, B, dev, torch.int64)
    k = torch.where((k <= 0) | (k > V), V, k)
    values, order = values.sort(dim=1, descending=True, stable=True)
    weight = torch.where(values == top, 0.0, values.double() - top.double())
    weight = torch.where(values == -math.inf, 0.0, (weight / torch.where(T > 0, T, 1.0)).exp())
    weight = torch.where(index < k, weight, 0.0)
    before = weight.cumsum(1) - weight
    weight = torch.where((before < p * weight.sum(1, keepdim=True)) | (index == 0) | (p >= 1), weight, 0.0)
    weight = torch.where(weight >= least, weight, 0.0)
    weight = torch.zeros_like(weight).scatter_(1, order, weight)
    total = weight.cumsum(1)
    token = (total <= u.double()[:, None] * total[:, -1:]).sum(1)
    last = torch.where(weight > 0, index, -1).amax(1)
    token = torch.minimum(token, last)
    token = torch.where(T[:, 0] > 0, token, greedy)
    return torch.where(top[:, 0] == -math.inf, -1, token)


def run(state):
    s = state
    op = s["op"]
    if op == "norm_rope":
        if own:
            return _framework().rope.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                                  positions=s["positions"], eps=s["eps"], interleaved=s["interleaved"])
        at = s["positions"].long()
        cos, sin = s["cos"][at], s["sin"][at]
        return (_plain_norm_rope(s["q"], s["wq"], cos, sin, s["eps"], s["interleaved"]),
                _plain_norm_rope(s["k"], s["wk"], cos, sin, s["eps"], s["interleaved"]))
    if op == "norm_append":
        if own:
            q = _framework().attention.qk_norm_rope_append(
                s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"], s["cos"], s["sin"],
                s["wq"], s["wk"], eps=s["eps"], interleaved=s["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        at = s["positions"].long()
        cos, sin = s["cos"][at], s["sin"][at]
        q = _plain_norm_rope(s["q"], s["wq"], cos, sin, s["eps"], s["interleaved"])
        block = s["k_cache"].shape[2]
        page, pos = s["slots"] // block, s["slots"] % block
        s["k_cache"][page, :, pos] = _plain_norm_rope(s["k"], s["wk"], cos, sin, s["eps"], s["interleaved"])
        s["v_cache"][page, :, pos] = s["v"]
        return q, s["k_cache"], s["v_cache"]
    if op == "fork":
        # the step's table and counts are made anew, so that every pass begins with the same pool
        table, counts = s["table"].clone(), s["counts"].clone()
        if own:
            kv = _framework().kv_cache
            child, moves = kv.kv_fork(table, s["lens"], s["parents"], counts, s["block"])
            kv.kv_copy_pages(s["k"], s["v"], moves)
            kv.kv_free(table, s["rows"], counts)
        else:
            child, src, dst, rows = _plain_fork(table, s["lens"], s["parents"], counts, s["block"])
            _plain_copy(s["k"] + s["v"], src, dst, rows)
            _plain_free(table, s["rows"], counts)
        return child, table, counts, s["k"], s["v"]
    if op == "compact":
        table, counts = s["table"].clone(), s["counts"].clone()
        if own:
            kv = _framework().kv_cache
            page_map, moves = kv.kv_compact(table, counts)
            kv.kv_copy_pages(s["k"], s["v"], moves)
        else:
            page_map, src, dst = _plain_compact(table, counts)
            _plain_copy(s["k"] + s["v"], src, dst)
        return page_map, table, counts, s["k"], s["v"]
    if own:
        return _framework().softmax.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                                  top_p=s["top_p"], min_p=s["min_p"])
    return _plain_sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "float32" else 2
    if op in ("norm_append", "norm_rope"):
        if op == "norm_append":
            n = int(_new_tokens(case).sum())
            rows, moved = min(n, case["ctx"] + abs(case["new"])), case["hq"] + 2 * case["hkv"]
        else:
            n, moved = case["tokens"], case["hq"] + case["hkv"]
            rows = case["ctx"] * -math.expm1(-n / case["ctx"])  # distinct positions among n drawn ones
        te = 4 if case["tables"] == "float32" else e
        # half of a table's row is a copy of the other half
        return {"bytes": int(2 * n * moved * case["dim"] * e + rows * case["dim"] * te + n * 12),
                "flops": int(n * (case["hq"] + case["hkv"]) * case["dim"] * 7)}
    if op == "sample":
        return {"bytes": int(case["rows"] * (case["vocab"] * e + 28)), "flops": int(case["rows"] * case["vocab"] * 4)}
    page = case["hkv"] * case["block"] * case["dim"] * e * 2 * case["layers"]
    if op == "fork":
        entries = (case["parents"] + case["children"]) * (case["ctx"] / 2 / case["block"])
        part = case["children"] * (case["block"] - 1) / case["block"]  # those with a part-filled last page
        return {"bytes": int(2 * part * page / 2 + entries * 24 + case["pool"] * 4), "flops": int(entries)}
    movers = case["pool"] * case["free"] * (1 - case["free"])
    return {"bytes": int(2 * movers * page + case["pool"] * (4 + 4 + 8 + 16)), "flops": case["pool"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def _exact_rotated(x, w, cos, sin, eps, interleaved):
    """The pairs of a head as complex numbers, times the table's."""
    x = x.double()
    half = x.shape[-1] // 2
    x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + eps).sqrt() * w.double()
    if interleaved:
        z = torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous())
        turn = torch.complex(cos[:, 0::2].double().contiguous(), sin[:, 0::2].double().contiguous())
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
        turn = torch.complex(cos[:, :half].double().contiguous(), sin[:, :half].double().contiguous())
    z = z * turn[:, None]
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)


def _exact_tokens(s):
    """Row by row on the host: the kept set as a list, the draw by a search in its running sum."""
    logits = s["logits"].double().cpu().numpy()
    B, V = logits.shape
    u = s["u"].double().cpu().numpy()
    row_of = lambda v, t: v.cpu().numpy() if torch.is_tensor(v) else np.full(B, v, dtype=t)  # noqa: E731
    T, P = row_of(s["temperature"], np.float32), row_of(s["top_p"], np.float32)
    K, M = row_of(s["top_k"], np.int64), row_of(s["min_p"], np.float32)
    tokens = np.empty(B, dtype=np.int64)
    for b in range(B):
        x = logits[b]
        if not T[b] > 0:
            tokens[b] = np.argmax(x)
            continue
        best = np.argsort(-x, kind="stable")
        if 0 < K[b] < V:
            best = best[:K[b]]
        w = np.exp((x[best] - x[best[0]]) / np.float64(T[b]))
        run_sum = np.cumsum(w)
        n = len(best)
        if P[b] < 1:
            n = max(1, int(np.count_nonzero(run_sum - w < np.float64(P[b]) * run_sum[-1])))
        n = min(n, int(np.count_nonzero(w >= min(np.float64(M[b]), 1.0))))
        kept = np.sort(best[:n])
        w = np.exp((x[kept] - x[best[0]]) / np.float64(T[b]))
        run_sum = np.cumsum(w)
        tokens[b] = kept[min(n - 1, int(np.searchsorted(run_sum, u[b] * run_sum[-1], side="right")))]
    return torch.from_numpy(tokens)


def _exact_fork(s):
    """Child by child on the host, with a list of the free pages; then page by page in the caches, which only moves."""
    table, counts, lens = s["table"].cpu().numpy().copy(), s["counts"].cpu().numpy().copy(), s["lens"].cpu().numpy()
    block, free = s["block"], [int(page) for page in np.flatnonzero(counts == 0)[::-1]]
    child = np.full((len(s["parents"]), table.shape[1]), -1, dtype=np.int64)
    for i, p in enumerate(s["parents"].cpu().numpy()):
        full, rest = divmod(int(lens[p]), block)
        child[i, :full] = table[p, :full]
        counts[table[p, :full]] += 1
        if rest:
            page = free.pop()
            counts[page] = 1
            child[i, full] = page
            for cache in s["k"] + s["v"]:
                cache[page, :, :rest] = cache[int(table[p, full]), :, :rest]
    for r in s["rows"].cpu().numpy():
        counts[table[r][table[r] >= 0]] -= 1
        table[r] = -1
    return torch.from_numpy(child), torch.from_numpy(table), torch.from_numpy(counts), s["k"], s["v"]


def _exact_compact(s):
    """Two fingers on the host: the last live page into the first hole, until they meet."""
    counts = s["counts"].cpu().numpy().copy()
    page_map = np.where(counts > 0, np.arange(len(counts)), -1)
    low, high, src, dst = 0, len(counts) - 1, [], []
    while True:
        while low < len(counts) and counts[low] > 0:
            low += 1
        while high >= 0 and counts[high] == 0:
            high -= 1
        if low >= high:
            break
        counts[low], counts[high], page_map[high] = counts[high], 0, low
        src.append(high)
        dst.append(low)
    table = s["table"].cpu().numpy()
    table = np.where(table >= 0, page_map[np.maximum(table, 0)], table)
    for cache in s["k"] + s["v"]:
        cache[dst] = cache[src]
    return torch.from_numpy(page_map), torch.from_numpy(table), torch.from_numpy(counts), s["k"], s["v"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fork":
        return _exact_fork(s)
    if case["op"] == "compact":
        return _exact_compact(s)
    if case["op"] == "sample":
        return _exact_tokens(s)
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    q = _exact_rotated(s["q"], s["wq"], cos, sin, s["eps"], s["interleaved"])
    k = _exact_rotated(s["k"], s["wk"], cos, sin, s["eps"], s["interleaved"])
    if case["op"] == "norm_rope":
        return q, k
    block = s["k_cache"].shape[2]
    page, pos = s["slots"] // block, s["slots"] % block
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache[page, :, pos] = k
    v_cache[page, :, pos] = s["v"].double()
    return q, k_cache, v_cache
