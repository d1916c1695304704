"""The batched-serving operators over an 8-bit paged KV cache: what they compute, on which shapes, and what it costs at least.

Four operators make one step of a batch of requests: ``tables`` (block table and slot map from the request lengths), ``append``
(RoPE, then K and V into the cache as 8-bit codes with a scale per block of tokens and head), ``attend`` (attention that reads
that cache) and ``sample`` (temperature, top-k, top-p and min-p from given uniform numbers).

``run`` computes them in plain torch, in 32 bits and rounded once, or through the framework's calls when ``own`` is set.
``exact`` restates each definition in 64 bits, request by request.
"""
import math
import random

import torch

own = False

DEV = "cuda"
QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
REAL = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SMALLEST_SCALE = 2.0 ** -100  # a scale below this is stored as zero
WEIGHT_ONE = 2.0 ** 31        # the weight of the most probable token


# ---- the cases ------------------------------------------------------------------

def listed():
    return [
        # One decode step's bookkeeping for 64 requests of up to 8192 tokens: every call of a serving loop.
        {"name": "tables_step", "op": "tables", "requests": 64, "context": 8191, "query": 1, "ragged": False, "block": 64, "lengths": 1},
        # A wave of 1000 ragged prompts admitted at once, some with cached prefixes.
        {"name": "tables_prompts", "op": "tables", "requests": 1000, "context": 700, "query": 511, "ragged": True, "block": 16, "lengths": 2},
        # A decode step's cache write for 64 requests, 70B-shaped heads: one token each, blocks partly filled.
        {"name": "append_step", "op": "append", "requests": 64, "context": 200, "query": 1, "ragged": False, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 64, "cache": "e4m3", "dtype": "f16", "rope": True, "lengths": 3},
        # Five ragged prompts, about 20 thousand tokens, 7B-shaped heads, blocks of 16.
        {"name": "append_prompts", "op": "append", "requests": 5, "context": 77, "query": 8111, "ragged": True, "heads": 32, "kv_heads": 32,
         "dim": 128, "block": 16, "cache": "int8", "dtype": "bf16", "rope": True, "lengths": 4},
        # The 7B-shaped decode step at 512 positions, one request: latency.
        {"name": "attend_one", "op": "attend", "requests": 1, "context": 512, "query": 1, "ragged": False, "heads": 32, "kv_heads": 32,
         "dim": 128, "block": 64, "cache": "int8", "dtype": "f16", "lengths": 5},
        # A serving batch of 64 ragged requests up to 16384 tokens, 70B-shaped heads.
        {"name": "attend_batch", "op": "attend", "requests": 64, "context": 16384, "query": 1, "ragged": True, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 64, "cache": "e4m3", "dtype": "f16", "lengths": 6},
        # Two long documents: the work of one head has to be split over many SMs.
        {"name": "attend_long", "op": "attend", "requests": 2, "context": 131071, "query": 1, "ragged": False, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 64, "cache": "int8", "dtype": "bf16", "lengths": 7},
        # Five draft tokens a request to check at once, heads of 256 with 16 queries to a KV head, odd lengths.
        {"name": "attend_draft", "op": "attend", "requests": 33, "context": 2047, "query": 5, "ragged": True, "heads": 32, "kv_heads": 2,
         "dim": 256, "block": 32, "cache": "e4m3", "dtype": "bf16", "lengths": 8},
        # Prompt chunks of up to 2048 tokens over what is cached already: matrix products on tensor cores.
        {"name": "attend_prompts", "op": "attend", "requests": 3, "context": 6000, "query": 2048, "ragged": True, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 64, "cache": "e4m3", "dtype": "f16", "lengths": 9},
        # One row of the 7B-shaped vocabulary with the usual three filters: latency.
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "f16", "filters": "k p", "lengths": 10},
        # 256 rows of a large vocabulary, every row with its own mix of filters, greedy rows among them.
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 131072, "dtype": "f16", "filters": "mixed", "lengths": 11},
        # Rollouts: the whole distribution, 32-bit logits, an odd vocabulary.
        {"name": "sample_rollout", "op": "sample", "rows": 48, "vocab": 50001, "dtype": "f32", "filters": "none", "lengths": 12},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))
    v = max(low, min(high, v))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "attend", "sample"])
    seed = rng.randrange(1 << 30)
    if op == "sample":
        rows = _spread(rng, 1, 256)
        return {"op": op, "rows": rows, "vocab": _spread(rng, 100, min(131072, 30_000_000 // rows)), "dtype": rng.choice(["f16", "bf16", "f32"]),
                "filters": rng.choice(["none", "k p", "p", "mixed", "mixed"]), "lengths": seed}
    block = rng.choice([16, 32, 64, 128])
    if op == "tables":
        query = _spread(rng, 1, 600)
        return {"op": op, "requests": _spread(rng, 1, min(1000, 280_000 // query)), "context": _spread(rng, 1, 8192), "query": query,
                "ragged": rng.random() < 0.7, "block": block, "lengths": seed}
    heads, kv_heads, dim = rng.choice([(32, 32, 128), (64, 8, 128), (32, 2, 256), (8, 8, 64), (32, 8, 64), (8, 1, 128), (12, 4, 128), (16, 4, 256)])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "cache": rng.choice(["int8", "e4m3"]),
            "dtype": rng.choice(["f16", "bf16"]), "ragged": rng.random() < 0.7, "lengths": seed}
    if op == "append":
        requests = _spread(rng, 1, 128)
        query = 1 if rng.random() < 0.4 else _spread(rng, 1, 8192 * 32 * 128 // (kv_heads * dim))
        query = max(1, min(query, 16384 // requests))
        return dict(case, requests=requests, context=_spread(rng, 1, 300), query=query, rope=rng.random() < 0.7)
    requests = _spread(rng, 1, 64)
    # at most the long case's cache and the prompt case's products
    context = _spread(rng, 1, max(1, min(131072, 260_000_000 // (requests * kv_heads * dim))))
    query = 1 if rng.random() < 0.5 else _spread(rng, 2, 2048)
    while requests * query * heads * dim * (context + query) > 5e10 and query > 1:
        query = (query + 1) // 2
    while requests * kv_heads * dim * (context + query) > 300_000_000:
        requests = max(1, requests // 2)
    return dict(case, requests=requests, context=context, query=query)


def _lengths(case):
    """(tokens cached before the step, new tokens) of each request: by the case alone."""
    r = random.Random(case["lengths"])
    n = case["requests"]
    if not case["ragged"]:
        return [case["context"]] * n, [case["query"]] * n
    context = [case["context"]] + [_spread(r, 1, case["context"]) for _ in range(n - 1)]
    query = [case["query"]] + [r.randint(1, case["query"]) for _ in range(n - 1)]
    return context, query


# ---- what a program has in hand -------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _paged(case, gen, spare=3):
    """Lengths, query starts and a block table over a shuffled pool."""
    context, query = _lengths(case)
    bs = case["block"]
    used = [-(-(c + n) // bs) for c, n in zip(context, query)]
    width = max(used) + 1
    pool = sum(used) + spare
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=DEV)
    mask = torch.arange(width, device=DEV)[None, :] < _ints(used)[:, None]
    table[mask] = order[: sum(used)]
    starts = [0]
    for n in query:
        starts.append(starts[-1] + n)
    return context, query, table, pool, starts


def _codes(case, pool, gen):
    """A cache as the write operator leaves it: normal values, some channels larger, most blocks near full range."""
    shape = (pool, case["kv_heads"], case["block"], case["dim"])
    top = QMAX[case["cache"]]
    channel = 0.15 + 0.2 * torch.rand(case["kv_heads"], 1, case["dim"], generator=gen, device=DEV, dtype=torch.float32)
    codes = torch.empty(shape, dtype=CODE[case["cache"]], device=DEV)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, pool, step):
        x = torch.randn((min(step, pool - i),) + shape[1:], generator=gen, device=DEV, dtype=torch.float32)
        x = (x * channel * top).clamp_(-top, top)
        codes[i:i + step] = (x.round_() if case["cache"] == "int8" else x).to(codes.dtype)
    scales = (4.0 / top) * torch.exp(0.3 * torch.randn(shape[:2], generator=gen, device=DEV, dtype=torch.float32))
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 1000003 + case["lengths"])
    s = {"op": case["op"]}
    if case["op"] == "sample":
        b, v = case["rows"], case["vocab"]
        # logits as a trained head gives them: a wide body and a few tokens that stand out
        x = 2.0 * torch.randn(b, v, generator=gen, device=DEV)
        hot = torch.randint(0, v, (b, 12), generator=gen, device=DEV)
        x.scatter_add_(1, hot, 4.0 + 6.0 * torch.rand(b, 12, generator=gen, device=DEV))
        x[:, v // 3] = -math.inf  # a token that a grammar forbids
        s["logits"] = x.to(REAL[case["dtype"]])
        s["uniforms"] = torch.rand(b, generator=gen, device=DEV)
        row = torch.arange(b, device=DEV)
        f = case["filters"]
        s["temperature"] = s["top_k"] = s["top_p"] = s["min_p"] = None
        if f == "none":
            s["temperature"] = torch.ones(b, device=DEV)
        else:
            s["temperature"] = 0.6 + 0.6 * torch.rand(b, generator=gen, device=DEV)
            s["top_p"] = 0.8 + 0.19 * torch.rand(b, generator=gen, device=DEV)
        if f == "k p":
            s["top_k"] = torch.full((b,), 40, dtype=torch.int32, device=DEV)
        if f == "mixed":
            s["top_k"] = torch.where(row % 3 == 0, 0, 1 + (row * 37) % 400).to(torch.int32)
            s["top_p"] = torch.where(row % 4 == 1, 1.0, s["top_p"])
            s["min_p"] = torch.where(row % 5 == 2, 0.02, 0.0).float()
            s["temperature"] = torch.where(row % 7 == 3, 0.0, s["temperature"])
        return s
    context, query, table, pool, starts = _paged(case, gen)
    total = starts[-1]
    bs = case["block"]
    s.update(block=bs, tokens=total)
    if case["op"] == "tables":
        held = _ints([-(-c // bs) for c in context])
        keep = torch.arange(table.shape[1], device=DEV)[None, :] < held[:, None]
        s["table"] = torch.where(keep, table, -1).to(torch.int32)
        taken = torch.zeros(pool, dtype=torch.bool, device=DEV)
        taken[table[keep].long()] = True
        free = torch.arange(pool, dtype=torch.int32, device=DEV)[~taken]
        # a queue of free blocks whose first two entries went out before
        s["free"] = torch.cat([free[-2:], free[torch.randperm(free.numel(), generator=gen, device=DEV)]])
        s["head"] = _ints([2])
        s.update(context=_ints(context), new=_ints(query))
        return s
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    dt = REAL[case["dtype"]]
    s["k_cache"], s["k_scale"] = _codes(case, pool, gen)
    s["v_cache"], s["v_scale"] = _codes(case, pool, gen)
    if case["op"] == "append":
        # the projections' output: q, k and v side by side in one row per token
        x = torch.randn(total, hq + 2 * hk, d, generator=gen, device=DEV).to(dt)
        s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        c, n, st = _ints(context, torch.int64), _ints(query, torch.int64), _ints(starts, torch.int64)
        req = torch.repeat_interleave(torch.arange(case["requests"], device=DEV), n, output_size=total)
        s["positions"] = c[req] + torch.arange(total, device=DEV) - st[req]
        s["slots"] = table[req, s["positions"] // bs].long() * bs + s["positions"] % bs
        s["freqs"] = None
        if case["rope"]:
            inv = 10000.0 ** (-torch.arange(0, d, 2, device=DEV).float() / d)
            ang = torch.outer(torch.arange(max(a + b for a, b in zip(context, query)), device=DEV).float(), inv)
            s["freqs"] = torch.stack([ang.cos(), ang.sin()], -1).contiguous()
        return s
    s["q"] = (1.5 * torch.randn(total, hq, d, generator=gen, device=DEV)).to(dt)
    s.update(table=table, seq_lens=_ints([a + b for a, b in zip(context, query)]), starts=_ints(starts), max_query=max(query),
             max_seq=max(a + b for a, b in zip(context, query)), scale=1.0 / math.sqrt(d))
    s["workspace"] = torch.zeros(64 << 20, dtype=torch.uint8, device=DEV)  # kept by a serving loop from step to step
    return s


# ---- one pass -------------------------------------------------------------------

def run(state):
    s = state
    if own:
        from gdsllm_b200 import paged, sampling
        if s["op"] == "tables":
            t = paged.build_tables(s["context"], s["new"], s["table"], s["free"], s["head"], s["block"], s["tokens"])
            return {"table": s["table"], "seq_lens": t.seq_lens, "starts": t.query_starts, "positions": t.positions, "slots": t.slots, "head": t.free_head}
        if s["op"] == "append":
            q = paged.append_kv8(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                 q=None if s["freqs"] is None else s["q"], freqs=s["freqs"], positions=s["positions"])
            return _appended(s, q)
        if s["op"] == "attend":
            return paged.attend_kv8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"], s["starts"],
                                    s["max_query"], s["max_seq"], softmax_scale=s["scale"], workspace=s["workspace"])
        tokens, logprobs = sampling.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    return {"tables": _tables, "append": _append, "attend": _attend, "sample": _sample}[s["op"]](s)


def _appended(s, q):
    """The updated state: the codes as the cache holds them (a float8 code is its value, an int8 code is compared as a whole number) beside the scales."""
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if q is not None:
        out["q"] = q
    return out


def _tables(s):
    bs, table = s["block"], s["table"]
    seq = s["context"] + s["new"]
    held, after = (s["context"] + bs - 1) // bs, (seq + bs - 1) // bs
    need = after - held
    first = s["head"] + torch.cumsum(need, 0) - need
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (column >= held[:, None]) & (column < after[:, None])
    at = (first[:, None] + column - held[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    ends = torch.cumsum(s["new"], 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    i = torch.arange(s["tokens"], device=table.device)
    req = torch.searchsorted(ends, i, right=True)
    positions = s["context"][req] + i - starts[req]
    slots = table[req, positions // bs].long() * bs + positions % bs
    return {"table": table, "seq_lens": seq, "starts": starts, "positions": positions, "slots": slots, "head": (s["head"] + need.sum()).to(torch.int32)}


def _rotate(x, f):
    a, b = x.float()[..., 0::2], x.float()[..., 1::2]
    c, d = f[:, None, :, 0], f[:, None, :, 1]
    return torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2).to(x.dtype)


def _write(x, pages, offsets, first, page_of, cache, scale):
    """x [T, heads, dim] into the cache: the scale of every touched block, the codes held under it before, the new codes."""
    top = 448.0 if cache.dtype == torch.float8_e4m3fn else 127.0
    x = x.float()
    touched, begin = pages[first], offsets[first]
    most = torch.zeros(touched.numel(), x.shape[1], device=x.device).index_reduce_(0, page_of, x.abs().amax(-1), "amax")
    need = most * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)
    need = torch.where(need < SMALLEST_SCALE, 0.0, need)
    base = torch.where((begin == 0)[:, None], 0.0, scale[touched])
    new = torch.where(need <= base, base, torch.maximum(need, 2.0 * base))
    new = torch.where(torch.isfinite(most) & ~torch.isnan(base), new, math.nan)
    inverse = torch.where(new > 0, torch.reciprocal(new), 0.0)
    scale[touched] = new

    def code(v):
        v = torch.nan_to_num(v, 0.0).clamp(-top, top)
        return (torch.round(v) if cache.dtype == torch.int8 else v).to(cache.dtype)

    raw = cache.view(torch.uint8)
    old = raw[touched]
    before = torch.arange(cache.shape[2], device=x.device)[None, :] < begin[:, None]
    move = before[:, None, :, None] & (new != base)[:, :, None, None]
    moved = code(old.view(cache.dtype).float() * (base * inverse)[:, :, None, None])
    raw[touched] = torch.where(move, moved.view(torch.uint8), old)
    raw[pages, :, offsets] = code(x * inverse[page_of][:, :, None]).view(torch.uint8)


def _append(s):
    k, q = s["k"], None
    if s["freqs"] is not None:
        f = s["freqs"][s["positions"]]
        k, q = _rotate(k, f), _rotate(s["q"], f)
    bs = s["k_cache"].shape[2]
    pages, offsets = s["slots"] // bs, s["slots"] % bs
    change = torch.cat([torch.ones_like(pages[:1], dtype=torch.bool), pages[1:] != pages[:-1]])
    page_of = torch.cumsum(change, 0) - 1
    first = torch.nonzero(change).flatten()
    _write(k, pages, offsets, first, page_of, s["k_cache"], s["k_scale"])
    _write(s["v"], pages, offsets, first, page_of, s["v_cache"], s["v_scale"])
    return _appended(s, q)


def _gather(cache, scale, table, blocks):
    at = table[:, :blocks].clamp_min(0).long()
    x = cache.view(torch.uint8)[at].view(cache.dtype).float() * scale[at][..., None, None]  # [R, blocks, heads, block, dim]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    q, table, dev = s["q"], s["table"], s["q"].device
    r, (total, hq, d), hk, bs = table.shape[0], q.shape, s["k_cache"].shape[1], s["k_cache"].shape[2]
    blocks, most = -(-s["max_seq"] // bs), s["max_query"]
    k = _gather(s["k_cache"], s["k_scale"], table, blocks)
    starts, lens = s["starts"].long(), s["seq_lens"].long()
    n = starts[1:] - starts[:-1]
    i = torch.arange(most, device=dev)
    at = (starts[:-1, None] + i[None, :]).clamp_max(total - 1)
    x = q[at].float().view(r, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(r, hk, -1, d)
    scores = torch.matmul(x, k.transpose(2, 3)) * s["scale"]
    del k
    column = torch.arange(blocks * bs, device=dev)
    seen = column[None, None, :] <= (lens - n)[:, None, None] + i[None, :, None]
    seen &= column[None, None, :] < lens[:, None, None]
    scores = scores.view(r, hk, hq // hk, most, blocks * bs).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total_weight = scores.sum(-1, keepdim=True)
    v = _gather(s["v_cache"], s["v_scale"], table, blocks)
    v = torch.where(column[None, None, :, None] < lens[:, None, None, None], v, 0.0)
    o = torch.matmul(scores.flatten(2, 3), v).view(r, hk, hq // hk, most, d)
    o = torch.where(total_weight > 0, o / total_weight, 0.0)
    req = torch.repeat_interleave(torch.arange(r, device=dev), n, output_size=total)
    o = o.permute(0, 3, 1, 2, 4).reshape(r, most, hq, d)
    return o[req, torch.arange(total, device=dev) - starts[req]].to(q.dtype)


def _or(value, like, default):
    return torch.full_like(like, default) if value is None else value


def _sample(s):
    u = s["uniforms"]
    x = torch.nan_to_num(s["logits"].float(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    v = x.shape[1]
    t = _or(s["temperature"], u, 1.0)
    k = _or(s["top_k"], torch.zeros_like(u, dtype=torch.int32), 0)
    k = torch.where(t > 0, torch.where((k <= 0) | (k > v), v, k), 1)
    inverse = torch.where(t > 0, torch.reciprocal(t), 1.0)
    top = x.amax(1, keepdim=True)
    e = torch.where(x == top, 1.0, torch.exp((x - top) * inverse[:, None]))
    e = torch.where(x == -math.inf, 0.0, e)
    w = (e * WEIGHT_ONE).to(torch.int64)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    sorted_w = torch.gather(w, 1, order)
    keep = torch.arange(v, device=x.device)[None, :] < k[:, None]
    sorted_w = torch.where(keep, sorted_w, 0)
    before = torch.cumsum(sorted_w, 1) - sorted_w
    limit = _or(s["top_p"], u, 1.0).double()[:, None] * sorted_w.sum(1, keepdim=True).double()
    keep &= (before.double() < limit) & (torch.gather(e, 1, order) >= _or(s["min_p"], u, 0.0)[:, None])
    keep[:, 0] = True
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(1, order, keep)
    w = torch.where(kept, w, 0)
    sums = torch.cumsum(w, 1)
    whole = sums[:, -1]
    target = torch.minimum((u.double() * whole.double()).to(torch.int64), whole - 1)
    tokens = (sums <= target[:, None]).sum(1).clamp_max(v - 1)
    p = torch.gather(w, 1, tokens[:, None])[:, 0].double() / whole.double()
    empty = whole == 0
    return {"tokens": torch.where(empty, -1, tokens), "logprobs": torch.where(empty, -math.inf, torch.log(p.float()))}


# ---- the definitions in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None  # whole numbers
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)


def _exact_append(case, s):
    """Block by block on the host's order of tokens; the key is rounded to its own type after the rotation, as the definition says."""
    q = None
    k = s["k"].double()
    if s["freqs"] is not None:
        z = torch.view_as_complex(s["freqs"].double())[s["positions"]][:, None, :]

        def turn(x):
            x = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
            return torch.view_as_real(x * z).reshape(x.shape[0], x.shape[1], -1)

        k, q = turn(s["k"]).to(s["k"].dtype).double(), turn(s["q"])
    bs = case["block"]
    top = QMAX[case["cache"]]
    slots = s["slots"].tolist()
    out = {}
    for name, x in (("k", k), ("v", s["v"].double())):
        cache, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        i = 0
        while i < len(slots):
            j = i
            while j < len(slots) and slots[j] // bs == slots[i] // bs:
                j += 1
            page, begin = slots[i] // bs, slots[i] % bs
            need = x[i:j].abs().amax((0, 2)) / top
            base = scale[page] if begin else torch.zeros_like(need)
            new = torch.where(need <= base, base, torch.maximum(need, 2 * base))
            cache[page, :, :begin] *= torch.where(new > 0, base / new, 1.0)[:, None, None]
            cache[page, :, begin:begin + j - i] = (x[i:j] / new[None, :, None]).transpose(0, 1)
            scale[page] = new
            i = j
        out[name + "_cache"] = cache if case["cache"] == "e4m3" else None
        out[name + "_scale"] = scale
    if q is not None:
        out["q"] = q
    return out


def _exact_attend(case, s):
    total, hq, d = s["q"].shape
    hk, bs = case["kv_heads"], case["block"]
    out = torch.zeros(total, hq, d, dtype=torch.float64, device=DEV)
    context, query = _lengths(case)
    at = 0
    for r, (c, n) in enumerate(zip(context, query)):
        rows = s["table"][r, :-(-(c + n) // bs)].long()
        hidden = torch.arange(c + n, device=DEV)[None, :] > c + torch.arange(n, device=DEV)[:, None]
        for h in range(hk):
            k = (s["k_cache"].view(torch.uint8)[rows, h].view(s["k_cache"].dtype).double() * s["k_scale"][rows, h].double()[:, None, None]).reshape(-1, d)[:c + n]
            v = (s["v_cache"].view(torch.uint8)[rows, h].view(s["v_cache"].dtype).double() * s["v_scale"][rows, h].double()[:, None, None]).reshape(-1, d)[:c + n]
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            a = (s["q"][at:at + n, heads].double().transpose(0, 1) @ k.T) / math.sqrt(d)
            out[at:at + n, heads] = (torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v).transpose(0, 1)
        at += n
    return out


def _exact_sample(case, s):
    """Row by row. The weights are whole by definition, so the choice is exact; the log-probability is taken in 64 bits."""
    logprobs = []
    for b in range(case["rows"]):
        def of(name, default):
            return default if s[name] is None else s[name][b].item()
        x = s["logits"][b].float()
        t, k = of("temperature", 1.0), of("top_k", 0)
        greedy = t <= 0
        z = (x - x.max()) * (1.0 if greedy else torch.reciprocal(s["temperature"][b]))
        e = torch.exp(z)
        w = torch.floor(e.double() * WEIGHT_ONE)
        index = torch.sort(x, descending=True, stable=True).indices
        k = 1 if greedy else k if 0 < k < x.numel() else x.numel()
        index = index[:k]
        run_sum = torch.cumsum(w[index], 0)
        keep = torch.cat([torch.zeros_like(run_sum[:1]), run_sum[:-1]]) < of("top_p", 1.0) * run_sum[-1]
        keep &= e[index] >= of("min_p", 0.0)
        keep[0] = True
        index = torch.sort(index[keep]).values
        run_sum = torch.cumsum(w[index], 0)
        target = torch.clamp(torch.floor(s["uniforms"][b].double() * run_sum[-1]), max=run_sum[-1] - 1)
        chosen = torch.searchsorted(run_sum, target.reshape(1), right=True)[0]
        logprobs.append(torch.log(w[index[chosen]] / run_sum[-1]))
    return {"tokens": None, "logprobs": torch.stack(logprobs)}


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 32, "flops": 4 * n}
    context, query = _lengths(case)
    total, requests, bs = sum(query), case["requests"], case["block"]
    if case["op"] == "tables":
        fresh = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(context, query))
        return {"bytes": 16 * total + 8 * fresh + 16 * requests, "flops": 0}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        touched = sum((c + n - 1) // bs - c // bs + 1 for c, n in zip(context, query))
        moved = total * hk * d * 2 * (2 + 1) + touched * hk * 16 + 8 * total
        if case["rope"]:
            moved += total * (hq * d * 4 + d * 4)
        return {"bytes": moved, "flops": 4 * total * hk * d + (3 * total * (hq + hk) * d if case["rope"] else 0)}
    tokens = sum(c + n for c, n in zip(context, query))
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, query))
    blocks = sum(-(-(c + n) // bs) for c, n in zip(context, query))
    return {"bytes": tokens * hk * d * 2 + blocks * (hk * 8 + 4) + total * hq * d * 4 + requests * 8, "flops": 4 * d * hq * pairs}
