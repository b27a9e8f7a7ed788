"""Measured cases of the serving operators around an 8-bit paged KV cache.

Four operators, each computed either in a plain form (elementary torch operations in
32 bits, rounded once at the end) or, with ``own`` true, by this package's kernels:

* ``maps``   - block tables, slot maps and positions of a round from request lengths
* ``norm``   - RMS norm of every query and key head with the position rotation in the same
  pass, and (``store`` other than "none") the K/V rows written into the paged cache
* ``tree``   - attention of packed draft trees (one node: an ordinary decode step) over the
  8-bit paged cache
* ``commit`` - accepted nodes' 8-bit rows and their scales moved to their final slots

An 8-bit row is 128 or 64 e4m3 codes and one power-of-two scale (e8m0) per slot and KV
head: scale = 2^e with the smallest e such that the row's largest magnitude is at most
448 * 2^e.
"""
from __future__ import annotations

import math
from types import SimpleNamespace
import zlib

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6
_package = None


def _jb():
    """This package, loaded on first use from the repository's root."""
    global _package
    if _package is None:
        import __graft_entry__

        _package = __graft_entry__.load_package()
    return _package


# ---- cases ------------------------------------------------------------------------------
def _maps(name, requests, cached, new, block):
    return {"name": name, "op": "maps", "requests": requests, "cached_max": cached,
            "new_min": new[0], "new_max": new[1], "block": block}


def _norm(name, tokens, heads, kv_heads, dim, dtype, store):
    return {"name": name, "op": "norm", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "store": store, "block": 256}


def _tree(name, requests, context, nodes, kv_heads, groups, dim, dtype, block=256):
    return {"name": name, "op": "tree", "requests": requests, "ctx_min": context[0],
            "ctx_max": context[1], "nodes_min": nodes[0], "nodes_max": nodes[1],
            "kv_heads": kv_heads, "groups": groups, "dim": dim, "dtype": dtype, "block": block}


def _commit(name, slots, layers, kv_heads, dim):
    return {"name": name, "op": "commit", "slots": slots, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "block": 256}


def listed():
    return [
        # One decode round of 64 requests: every request adds one token, a few need a page.
        _maps("maps_decode_64", 64, 16384, (1, 1), 256),
        # A prefill round of many ragged prompts into fresh and half-filled pages.
        _maps("maps_prefill_509", 509, 700, (1, 1000), 256),
        # Seven requests decode one token each (Qwen3-8B heads); latency counts.
        _norm("norm_decode_7", 7, 32, 8, 128, "bf16", "fp8"),
        # The verification round of 32 requests with 64-node trees (Qwen3-8B heads).
        _norm("norm_verify_2048", 2048, 32, 8, 128, "bf16", "fp8"),
        # A prefill chunk of an odd length into the 8-bit cache.
        _norm("norm_prefill_16381", 16381, 32, 8, 128, "bf16", "fp8"),
        # 64-wide f16 heads with 7 queries for each key head, no cache (rotated K returned).
        _norm("norm_only_f16_d64", 4095, 14, 2, 64, "f16", "none"),
        # A small decode batch: one token for each of 5 requests, short contexts.
        _tree("tree_decode_5", 5, (1, 900), (1, 1), 8, 4, 128, "bf16"),
        # Long-context decode: one token for each of 16 requests.
        _tree("tree_decode_long", 16, (30000, 32768), (1, 1), 8, 4, 128, "bf16"),
        # The verification step of 32 requests, 2048-token contexts, 64-node trees.
        _tree("tree_verify_2048", 32, (2048, 2048), (64, 64), 8, 4, 128, "bf16"),
        # The ragged serving mix: contexts 512..16384, trees of 16 to 128 nodes.
        _tree("tree_serving_mix", 64, (512, 16384), (16, 128), 8, 4, 128, "bf16"),
        # A round's accepted nodes across the 36 layers of Qwen3-8B.
        _commit("commit_96", 96, 36, 8, 128),
        # A large batch's accepted nodes.
        _commit("commit_2000", 2000, 36, 8, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["maps", "norm", "norm", "tree", "tree", "tree", "commit"])
    if op == "maps":
        requests = _log(rng, 1, 509)
        new_max = _log(rng, 1, 1000)
        case = _maps("", requests, _log(rng, 1, 16384), (rng.randint(1, new_max), new_max),
                     rng.choice([16, 64, 256]))
    elif op == "norm":
        dim = rng.choice([64, 128, 128])
        kv_heads, groups = rng.choice([(8, 4), (2, 7), (4, 8), (1, 4), (3, 5), (8, 1)])
        case = _norm("", _log(rng, 1, 16000), kv_heads * groups, kv_heads, dim,
                     rng.choice(["bf16", "bf16", "f16"]), rng.choice(["fp8", "fp8", "same", "none"]))
    elif op == "tree":
        requests = _log(rng, 1, 64)
        ctx_max = _log(rng, 1, min(32768, 512000 // requests))
        ctx_min = _log(rng, 1, ctx_max)
        nodes_max = _log(rng, 1, max(1, min(200, 4000 // requests)))
        kv_heads, groups = rng.choice([(8, 4), (8, 4), (2, 7), (4, 8), (1, 4), (3, 5), (8, 1)])
        case = _tree("", requests, (ctx_min, ctx_max), (_log(rng, 1, nodes_max), nodes_max),
                     kv_heads, groups, rng.choice([64, 128, 128]),
                     rng.choice(["bf16", "bf16", "f16"]), rng.choice([64, 128, 256, 256]))
    else:
        case = _commit("", _log(rng, 1, 2000), rng.randint(1, 36), rng.choice([1, 2, 3, 8]),
                       rng.choice([64, 128]))
    del case["name"]
    return case


# ---- the 8-bit rows ---------------------------------------------------------------------
def _exponents(amax):
    """The smallest e with amax <= 448 * 2^e (0 for a row of zeros), within e8m0's range."""
    mantissa, power = torch.frexp(amax)  # amax = mantissa * 2^power, mantissa in [0.5, 1)
    e = power - 9 + (mantissa > 0.875).to(power.dtype)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-127, 127)


def _quantize(x):
    """(e4m3 codes [..., dim], e8m0 scales [...]) of fp32 rows; a row with a non-finite
    element gets the NaN scale."""
    amax = x.abs().amax(-1)
    finite = torch.isfinite(amax)
    e = _exponents(torch.where(finite, amax, torch.zeros_like(amax)))
    y = torch.ldexp(torch.where(finite.unsqueeze(-1), x, torch.zeros_like(x)), -e.unsqueeze(-1))
    byte = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return y.to(E4M3), byte.view(E8M0)


def _fresh_pool(blocks, block, kv_heads, dim):
    codes = torch.zeros((blocks, block, kv_heads, dim), dtype=torch.uint8, device=DEVICE)
    scale = torch.full((blocks, kv_heads, block), 127, dtype=torch.uint8, device=DEVICE)
    return codes.view(E4M3), scale.view(E8M0)


# ---- inputs -----------------------------------------------------------------------------
def _spread(rng, lo, hi, n):
    """n whole numbers spread over the logarithm of [lo, hi]."""
    x = np.exp(rng.uniform(math.log(lo), math.log(hi + 0.49), size=n))
    return np.clip(np.rint(x).astype(np.int64), lo, hi)


def _lengths(case):
    """The case's own lengths (cached and new tokens of each request for "maps", prefix and
    nodes for "tree"): another seed permutes them among the requests, so that every seed
    has the same totals."""
    own_seed = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode())
    rng, n = np.random.default_rng(own_seed), case["requests"]
    if case["op"] == "maps":
        cached = _spread(rng, 1, case["cached_max"], n)
        cached[rng.random(n) < 0.1] = 0  # new requests
        return cached, rng.integers(case["new_min"], case["new_max"] + 1, size=n)
    prefix = _spread(rng, case["ctx_min"], case["ctx_max"], n)
    if n > 2 and case["ctx_min"] < case["ctx_max"]:
        prefix[1] = 0  # a tree over an empty prefix
    return prefix, _spread(rng, case["nodes_min"], case["nodes_max"], n)


def _dev(a, dtype):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).to(DEVICE)


def _prepare_maps(case, rng):
    requests, block = case["requests"], case["block"]
    cached, new = (rng.permutation(x) for x in _lengths(case))
    have, need = -(-cached // block), -(-(cached + new) // block)
    width = (case["cached_max"] + case["new_max"]) // block + 2
    pages = rng.permutation(int(need.sum()) + 7)
    table = np.full((requests, width), -1, dtype=np.int64)
    used = 0
    for r in range(requests):
        table[r, :have[r]] = pages[used:used + have[r]]
        used += int(have[r])
    total = int(new.sum())
    return SimpleNamespace(
        tables=_dev(table, torch.int32), cached=_dev(cached, torch.int32),
        new=_dev(new, torch.int32), free=_dev(pages[used:], torch.int32), block=block,
        # A graph's padded length: the round's tokens rounded up.
        capacity=-(-total // 8) * 8)


def _prepare_norm(case, gen, rng):
    n, hq, hk, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    dtype, block = DTYPES[case["dtype"]], case["block"]
    # One QKV projection's output; q, k and v are views of its rows.
    qkv = torch.randn((n, (hq + 2 * hk) * dim), generator=gen, device=DEVICE).mul_(1.3).to(dtype)
    q = qkv[:, :hq * dim].view(n, hq, dim)
    k = qkv[:, hq * dim:(hq + hk) * dim].view(n, hk, dim)
    v = qkv[:, (hq + hk) * dim:].view(n, hk, dim)
    weight = [(1 + 0.2 * torch.randn(dim, generator=gen, device=DEVICE)).to(dtype) for _ in "qk"]
    max_position = 40960
    freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    angle = torch.arange(max_position, dtype=torch.float64, device=DEVICE)[:, None] * freq
    cache = torch.cat([angle.cos(), angle.sin()], -1).float()
    positions = torch.randint(0, max_position, (n,), generator=gen, device=DEVICE)
    s = SimpleNamespace(q=q, k=k, v=v, qw=weight[0], kw=weight[1], positions=positions,
                        cache=cache, store=case["store"], k_pool=None, v_pool=None,
                        k_scale=None, v_scale=None, slots=None, block=block)
    if case["store"] != "none":
        blocks = -(-n // block) + 2
        slots = torch.randperm(blocks * block, generator=gen, device=DEVICE)[:n]
        if n > 4:
            slots[n // 2] = -1  # a padding token of a captured graph
        s.slots = slots
        if case["store"] == "fp8":
            s.k_pool, s.k_scale = _fresh_pool(blocks, block, hk, dim)
            s.v_pool, s.v_scale = _fresh_pool(blocks, block, hk, dim)
        else:
            s.k_pool, s.v_pool = (torch.zeros((blocks, block, hk, dim), dtype=dtype, device=DEVICE)
                                  for _ in "kv")
    return s


def _tree_layout(case, rng):
    """(prefix lengths, parents of each tree, page order, tables, node slots) on the host."""
    requests, block = case["requests"], case["block"]
    prefix, nodes = (rng.permutation(x) for x in _lengths(case))
    parents = []
    for t in nodes:
        p = np.full(int(t), -1, dtype=np.int64)
        for i in range(1, int(t)):
            p[i] = rng.integers(max(0, i - 8), i)
        parents.append(p)
    have = -(-prefix // block)
    scratch = -(-int(nodes.sum()) // block)
    order = rng.permutation(int(have.sum()) + scratch + 3)
    width = max(1, int(have.max()))
    table = np.full((requests, width), -1, dtype=np.int64)
    used = 0
    for r in range(requests):
        table[r, :have[r]] = order[used:used + have[r]]
        used += int(have[r])
    pool_slots = (order[used:used + scratch, None] * block + np.arange(block)).reshape(-1)
    slots = pool_slots[rng.permutation(pool_slots.size)[:int(nodes.sum())]]
    return prefix, parents, order.size, table, slots


def _visible(parents):
    """[T, T]: node j sees itself and its ancestors."""
    t = len(parents)
    m = np.zeros((t, t), dtype=bool)
    for j in range(t):
        if parents[j] >= 0:
            m[j] = m[parents[j]]
        m[j, j] = True
    return m


def _pool_rows(gen, blocks, block, kv_heads, dim, std):
    """A layer's K or V cache after prefill: normal rows, a few channels and tokens larger."""
    channel = torch.ones(dim, device=DEVICE)
    channel[torch.randint(0, dim, (3,), generator=gen, device=DEVICE)] = 4.0
    codes, scale = _fresh_pool(blocks, block, kv_heads, dim)
    for b in range(0, blocks, 512):
        e = min(blocks, b + 512)
        x = torch.randn((e - b, block, kv_heads, dim), generator=gen, device=DEVICE)
        x *= channel
        x *= std * torch.exp(0.5 * torch.randn(x.shape[:-1], generator=gen, device=DEVICE))[..., None]
        c, s = _quantize(x)
        codes.view(torch.uint8)[b:e] = c.view(torch.uint8)
        scale.view(torch.uint8)[b:e] = s.view(torch.uint8).transpose(1, 2)
    return codes, scale


def _prepare_tree(case, gen, rng):
    prefix, parents, blocks, table, slots = _tree_layout(case, rng)
    counts = np.array([len(p) for p in parents])
    cu = np.concatenate([[0], np.cumsum(counts)])
    bias = np.concatenate([np.where(_visible(p), 0.0, -np.inf).reshape(-1) for p in parents])
    hk, groups, dim, dtype = case["kv_heads"], case["groups"], case["dim"], DTYPES[case["dtype"]]
    total = int(counts.sum())
    meta = SimpleNamespace(
        cu_seqlens_q=_dev(cu, torch.int32),
        query_to_request=_dev(np.repeat(np.arange(len(counts)), counts), torch.int32),
        query_local_row=_dev(np.concatenate([np.arange(c) for c in counts]), torch.int32),
        prefix_lens=_dev(prefix, torch.int32), node_counts=_dev(counts, torch.int32),
        block_tables=_dev(table, torch.int32), tree_slots=_dev(slots, torch.int64),
        qq_bias=_dev(bias, torch.float32),
        qq_bias_offsets=_dev(np.concatenate([[0], np.cumsum(counts.astype(np.int64) ** 2)]),
                             torch.int64),
        block_size=case["block"], num_requests=len(counts), total_queries=total,
        node_counts_host=tuple(int(c) for c in counts))
    q = torch.randn((total, hk * groups, dim), generator=gen, device=DEVICE).to(dtype)
    k_pool, k_scale = _pool_rows(gen, blocks, case["block"], hk, dim, 1.0)
    v_pool, v_scale = _pool_rows(gen, blocks, case["block"], hk, dim, 1.3)
    return SimpleNamespace(q=q, k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale,
                           meta=meta, scale=dim ** -0.5, groups=groups,
                           longest=int(prefix.max()), widest=int(counts.max()))


def _prepare_commit(case, gen, rng):
    n, layers, hk, dim, block = (case[k] for k in ("slots", "layers", "kv_heads", "dim", "block"))
    blocks = -(-2 * n // block) + 2
    pool = torch.randint(0, 127, (2, layers, blocks, block, hk, dim), generator=gen,
                         dtype=torch.uint8, device=DEVICE)
    scale = torch.randint(110, 130, (2, layers, blocks, hk, block), generator=gen,
                          dtype=torch.uint8, device=DEVICE)
    order = torch.randperm(blocks * block, generator=gen, device=DEVICE)
    return SimpleNamespace(pool=pool.view(E4M3), scale=scale.view(E8M0), source=order[:n].clone(),
                           destination=order[n:2 * n].clone(), block=block)


def prepare(case, seed):
    rng = np.random.default_rng([seed, 17])
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 11)
    if case["op"] == "maps":
        s = _prepare_maps(case, rng)
    elif case["op"] == "norm":
        s = _prepare_norm(case, gen, rng)
    elif case["op"] == "tree":
        s = _prepare_tree(case, gen, rng)
    else:
        s = _prepare_commit(case, gen, rng)
    s.op = case["op"]
    return s


# ---- one pass ---------------------------------------------------------------------------
def _run_maps(s):
    if own:
        m = _jb().build_request_maps(s.tables, s.cached, s.new, s.free, s.block,
                                     max_tokens=s.capacity)
        return (m.block_tables, m.slot_mapping, m.positions, m.token_to_request, m.cu_seqlens,
                m.context_lens, m.pages_taken)
    cached, new, block = s.cached.long(), s.new.long(), s.block
    lens = cached + new
    have, need = (cached + block - 1) // block, (lens + block - 1) // block
    take = need - have
    first = take.cumsum(0) - take  # each request's first page of the free list
    column = torch.arange(s.tables.shape[1], device=s.tables.device)[None]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    at = first[:, None] + column - have[:, None]
    page = torch.where(at < s.free.numel(), s.free[at.clamp(0, s.free.numel() - 1)], -1)
    s.tables.copy_(torch.where(fresh, page, s.tables))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    token = torch.arange(s.capacity, device=s.tables.device)
    live = token < cu[-1]
    request = torch.where(live, torch.searchsorted(cu, token, right=True) - 1, 0)
    position = cached[request] + token - cu[request]
    col = (position // block).clamp(max=s.tables.shape[1] - 1)
    page = s.tables[request, col].long()
    slot = torch.where(live & (page >= 0), page * block + position % block, -1)
    return (s.tables, slot, torch.where(live, position, 0),
            torch.where(live, request, -1).int(), cu.int(), lens.int(), take.sum().int().reshape(1))


def _normed_rotated(x, weight, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_norm(s):
    if own:
        jb = _jb()
        if s.store == "none":
            return jb.qk_norm_rope(s.q, s.k, s.qw, s.kw, s.positions, s.cache, EPS)
        q = jb.qk_norm_rope_store(s.q, s.k, s.v, s.qw, s.kw, s.positions, s.cache, s.k_pool,
                                  s.v_pool, s.slots, EPS, k_scale=s.k_scale, v_scale=s.v_scale)
        return (q, s.k_pool, s.v_pool) + ((s.k_scale, s.v_scale) if s.store == "fp8" else ())
    cos, sin = s.cache[s.positions].float()[:, None].chunk(2, -1)
    q = _normed_rotated(s.q, s.qw, cos, sin).to(s.q.dtype)
    k = _normed_rotated(s.k, s.kw, cos, sin)
    if s.store == "none":
        return q, k.to(s.k.dtype)
    live = s.slots >= 0
    slots = s.slots[live]
    page, offset = slots // s.block, slots % s.block
    if s.store == "same":
        s.k_pool[page, offset] = k[live].to(s.k.dtype)
        s.v_pool[page, offset] = s.v[live]
        return q, s.k_pool, s.v_pool
    kc, ks = _quantize(k[live])
    vc, vs = _quantize(s.v[live].float())
    # 8-bit types are indexed as bytes.
    s.k_pool.view(torch.uint8)[page, offset] = kc.view(torch.uint8)
    s.v_pool.view(torch.uint8)[page, offset] = vc.view(torch.uint8)
    s.k_scale.view(torch.uint8)[page, :, offset] = ks.view(torch.uint8)
    s.v_scale.view(torch.uint8)[page, :, offset] = vs.view(torch.uint8)
    return q, s.k_pool, s.v_pool, s.k_scale, s.v_scale


def _key_slots(s):
    """([R, K] slot of every key position, [R, K] whether there is one)."""
    m, block = s.meta, s.meta.block_size
    length = s.longest + s.widest
    position = torch.arange(length, device=DEVICE)[None]
    prefix, count = m.prefix_lens.long()[:, None], m.node_counts.long()[:, None]
    column = (position // block).clamp(max=m.block_tables.shape[1] - 1)
    page = m.block_tables.long().gather(1, column.expand(m.num_requests, -1))
    node = m.cu_seqlens_q[:-1].long()[:, None] + position - prefix
    slot = torch.where(position < prefix, page * block + position % block,
                       m.tree_slots[node.clamp(0, m.total_queries - 1)])
    return slot, position < prefix + count, position - prefix


def _rows_of(pool, scale, slot, live, block):
    """fp32 rows [R, K, H, D] of the 8-bit cache at the live slots, zeros elsewhere."""
    slot = torch.where(live, slot, 0)
    page, offset = slot // block, slot % block
    codes = pool.view(torch.uint8)[page, offset].view(E4M3).float()
    factor = scale.view(torch.uint8)[page, :, offset].view(E8M0).float()
    return torch.where(live[..., None, None], codes * factor[..., None], 0.0)


def _run_tree(s):
    if own:
        return _jb().packed_tree_attention_fp8(s.q, s.k_pool, s.v_pool, s.k_scale, s.v_scale,
                                               s.meta, s.scale, s.groups)
    m = s.meta
    slot, live, node = _key_slots(s)
    k = _rows_of(s.k_pool, s.k_scale, slot, live, m.block_size)
    requests, keys, heads, dim = k.shape
    row, req = m.query_local_row.long(), m.query_to_request.long()
    q = s.q.new_zeros((requests, s.widest, heads, s.groups, dim), dtype=torch.float32)
    q[req, row] = s.q.view(-1, heads, s.groups, dim).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(requests, heads, s.widest * s.groups, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * s.scale
    del k
    # Row j of request r sees key n of its tree where the bias is zero and n <= j.
    j = torch.arange(s.widest, device=DEVICE)[None, :, None]
    n = node[:, None, :]
    count = m.node_counts.long()[:, None, None]
    at = (m.qq_bias_offsets[:-1][:, None, None] + j * count + n).clamp(0, m.qq_bias.numel() - 1)
    seen = (n < 0) | ((n <= j) & (n < count) & (j < count) & (m.qq_bias[at] == 0))
    seen = (seen & live[:, None, :]).repeat_interleave(s.groups, 1)[:, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    del score
    total = p.sum(-1, keepdim=True)
    v = _rows_of(s.v_pool, s.v_scale, slot, live, m.block_size)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    out = out.view(requests, heads, s.widest, s.groups, dim).permute(0, 2, 1, 3, 4)
    return out[req, row].reshape(s.q.shape).to(s.q.dtype)


def _run_commit(s):
    if own:
        _jb().copy_accepted_kv_fp8(s.pool, s.scale, s.source, s.destination, s.block)
        return s.pool, s.scale
    pool, scale = s.pool.view(torch.uint8), s.scale.view(torch.uint8)
    sp, so = s.source // s.block, s.source % s.block
    dp, do = s.destination // s.block, s.destination % s.block
    pool[:, :, dp, do] = pool[:, :, sp, so]
    flat = scale.transpose(3, 4)  # [2, layers, blocks, block, heads]
    flat[:, :, dp, do] = flat[:, :, sp, so]
    return s.pool, s.scale


def run(state):
    return {"maps": _run_maps, "norm": _run_norm, "tree": _run_tree,
            "commit": _run_commit}[state.op](state)


# ---- work and exact values --------------------------------------------------------------
def work(case):
    if case["op"] == "maps":
        # Lengths and free pages in; tables' new entries, slots, positions, owners out.
        cached, new = _lengths(case)
        pages = -(-(cached + new) // case["block"]) - -(-cached // case["block"])
        return {"bytes": int(new.sum() * (8 + 8 + 4) + case["requests"] * 16 + pages.sum() * 8),
                "flops": 0}
    if case["op"] == "norm":
        n, hq, hk, dim = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        size = 4 if case["dtype"] == "f32" else 2
        read = n * (hq + hk) * dim * size + n * (dim * 4 + 8)
        write = n * hq * dim * size
        if case["store"] == "none":
            write += n * hk * dim * size
        else:
            read += n * hk * dim * size + n * 8
            write += 2 * n * hk * (dim + 1 if case["store"] == "fp8" else dim * size)
        return {"bytes": read + write, "flops": n * (hq + hk) * dim * 8}
    if case["op"] == "tree":
        prefix, count = _lengths(case)
        nodes = count.sum()
        hk, groups, dim = case["kv_heads"], case["groups"], case["dim"]
        cache = (prefix.sum() + nodes) * hk * (dim + 1) * 2
        rows = nodes * hk * groups * dim * 2 * 2
        pairs = nodes * prefix.sum() / case["requests"] + (count * (count + 1)).sum() / 2
        return {"bytes": int(cache + rows), "flops": int(pairs * hk * groups * dim * 4)}
    n, layers, hk, dim = (case[k] for k in ("slots", "layers", "kv_heads", "dim"))
    return {"bytes": 2 * 2 * n * layers * hk * (dim + 1) + 16 * n, "flops": 0}


def _exact_norm(s):
    cos, sin = s.cache[s.positions].double()[:, None].chunk(2, -1)

    def rotate(x, w):
        x = x.double()
        x = w.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
        half = x.shape[-1] // 2
        return torch.cat([x[..., :half] * cos - x[..., half:] * sin,
                          x[..., half:] * cos + x[..., :half] * sin], -1)

    q, k = rotate(s.q, s.qw), rotate(s.k, s.kw)
    if s.store == "none":
        return q, k
    live = s.slots >= 0
    flat = s.slots[live]
    blocks = s.k_pool.shape[0]

    def pool_of(rows):
        """(values held, scales) of the rows in a pool of zeros with scale one."""
        out = torch.zeros((blocks * s.block,) + rows.shape[1:], dtype=torch.float64, device=DEVICE)
        if s.store == "same":
            out[flat] = rows[live]
            return out.view(blocks, s.block, *rows.shape[1:]), None
        x = rows[live]
        amax = x.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
        y = x / step
        # To the nearest e4m3 value, ties to even: spacing 2^(floor(log2|y|) - 3), 2^-9 at least.
        ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out[flat] = torch.round(y / ulp) * ulp
        scale = torch.ones((blocks * s.block,) + rows.shape[1:-1], dtype=torch.float64,
                           device=DEVICE)
        scale[flat] = step[..., 0]
        return (out.view(blocks, s.block, *rows.shape[1:]),
                scale.view(blocks, s.block, -1).transpose(1, 2).contiguous())

    (kp, ks), (vp, vs) = pool_of(k), pool_of(s.v.double())
    return (q, kp, vp) if s.store == "same" else (q, kp, vp, ks, vs)


def _exact_tree(s):
    """Request by request, every key by its slot, in 64 bits."""
    m, block = s.meta, s.meta.block_size
    k_codes, v_codes = s.k_pool.view(torch.uint8), s.v_pool.view(torch.uint8)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    cu, prefix = m.cu_seqlens_q.tolist(), m.prefix_lens.tolist()
    offsets = m.qq_bias_offsets.tolist()

    def rows(codes, scale, slot):
        c = codes.reshape(-1, *codes.shape[2:])[slot].view(E4M3).double()
        f = scale.view(torch.uint8)[slot // block, :, slot % block].double() - 127
        return c * torch.exp2(f)[..., None]

    for r in range(m.num_requests):
        lo, hi, p = cu[r], cu[r + 1], prefix[r]
        t = hi - lo
        pos = torch.arange(p, device=DEVICE)
        slot = torch.cat([m.block_tables[r].long()[pos // block] * block + pos % block,
                          m.tree_slots[lo:hi]])
        k, v = rows(k_codes, s.k_scale, slot), rows(v_codes, s.v_scale, slot)
        mask = torch.zeros((t, p + t), dtype=torch.float64, device=DEVICE)
        mask[:, p:] = m.qq_bias[offsets[r]:offsets[r + 1]].view(t, t).double()
        q = s.q[lo:hi].double().view(t, k.shape[1], s.groups, -1)
        for h in range(k.shape[1]):
            w = torch.einsum("tgd,kd->tgk", q[:, h], k[:, h]) * s.scale + mask[:, None]
            w = torch.softmax(w, -1)
            out[lo:hi, h * s.groups:(h + 1) * s.groups] = torch.einsum("tgk,kd->tgd", w, v[:, h])
    return out


def _exact_commit(s):
    """The values held: every row and scale read before any is written."""
    pool, scale = s.pool.float().double(), s.scale.float().double().transpose(3, 4).contiguous()
    for held in (pool, scale):
        rows = held.view(held.shape[0], held.shape[1], -1, *held.shape[4:])
        rows[:, :, s.destination] = rows[:, :, s.source].clone()
    return pool, scale.transpose(3, 4)


def exact(case, seed):
    if case["op"] == "maps":
        return None  # whole numbers
    s = prepare(case, seed)
    return {"norm": _exact_norm, "tree": _exact_tree, "commit": _exact_commit}[case["op"]](s)
