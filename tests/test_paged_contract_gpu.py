"""What the batched-serving calls promise beside their formulas: padded steps, given outputs, hints, launches that overlap."""
from __future__ import annotations

import math

import pytest
import torch

from gdsllm_b200 import capi, paged, sampling
from test_paged_gpu import CODE, attend_ref, ints, make_cache

pytestmark = pytest.mark.gpu


def step(cuda, lens, new, heads, kv_heads, dim, bs=16, kind="int8", seed=0):
    """(q, caches and scales, table, lengths, starts) of one step over a pool in order."""
    blocks = [-(-n // bs) for n in lens]
    kc, ks = make_cache(sum(blocks), kv_heads, bs, dim, kind, cuda, seed + 1)
    vc, vs = make_cache(sum(blocks), kv_heads, bs, dim, kind, cuda, seed + 2)
    ids = iter(range(sum(blocks)))
    table = ints([[next(ids) for _ in range(b)] + [-1] * (max(blocks) - b) for b in blocks], cuda)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], heads, dim, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).half()
    return q, (kc, vc, ks, vs), table, lens, starts


@pytest.mark.parametrize("heads,kv_heads,dim,new", [(8, 2, 64, [1, 3, 2]), (8, 2, 128, [40, 1, 7]), (16, 1, 256, [1, 1, 1]), (16, 1, 256, [9, 1, 1])])
@pytest.mark.parametrize("spare", [1, 77])
def test_padding_tokens_give_zeros(cuda, heads, kv_heads, dim, new, spare):
    """A step padded to a fixed number of tokens, as a captured graph has it: the places behind the last request hold no stale values."""
    q, cache, table, lens, starts = step(cuda, [100, 45, 300], new, heads, kv_heads, dim)
    want = paged.attend_kv8(q, *cache, table, ints(lens, cuda), ints(starts, cuda), max(new))
    padded = torch.cat([q, torch.full((spare, heads, dim), math.nan, dtype=q.dtype, device=cuda)])
    out = torch.full_like(padded, math.nan)
    paged.attend_kv8(padded, *cache, table, ints(lens, cuda), ints(starts, cuda), max(new), out=out)
    assert torch.equal(out[:starts[-1]], want) and not out[starts[-1]:].any()


def test_a_step_without_requests_gives_zeros(cuda):
    q, cache, table, lens, starts = step(cuda, [100], [3], 8, 2, 64)
    out = torch.full_like(q, math.nan)
    paged.attend_kv8(q, *cache, table[:0], ints([], cuda), ints([0], cuda), 3, out=out)
    assert not out.any()
    out.fill_(math.nan)
    paged.attend_kv8(q, *cache, table, ints(lens, cuda), ints([0, 0], cuda), 0, out=out)
    assert not out.any()
    out.fill_(math.nan)
    paged.attend_kv8(q, *cache, table, ints(lens, cuda), ints([0, 0], cuda), 1, out=out)
    assert not out.any()


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (16, 1, 128), (12, 1, 256)])
def test_lengths_that_the_host_was_not_told(cuda, heads, kv_heads, dim):
    """max_query_len chooses the kernel only, max_seq_len nothing: more tokens and longer requests than they say are right."""
    new = [1, 70, 3, 0]
    q, cache, table, lens, starts = step(cuda, [200, 300, 3, 5], new, heads, kv_heads, dim)
    want, bound = attend_ref(q, *cache, table, lens, starts, 1 / math.sqrt(dim), 2.0 ** -11)
    for longest in (1, 2, 4, 70):
        ws = paged.attend_workspace(4, longest, heads, kv_heads, dim, cuda)
        for seq in (None, 0, 7, 300):
            got = paged.attend_kv8(q, *cache, table, ints(lens, cuda), ints(starts, cuda), longest, seq, workspace=ws)
            assert bool(((got.double() - want).abs() <= bound).all())
    assert capi.device_error(0) == 0


def test_given_outputs(cuda):
    """``out``, ``q_out``, ``tokens`` and ``logprobs`` are filled and returned, with the bits of a call that makes its own."""
    bs, heads, hk, dim, requests = 16, 4, 2, 64, 3
    context, new = ints([5, 16, 40], cuda), ints([1, 3, 1], cuda)
    free = torch.arange(20, dtype=torch.int32, device=cuda)
    before = ints([[10, -1, -1, -1], [11, -1, -1, -1], [12, 13, 14, -1]], cuda)
    tables = [before.clone(), before.clone()]
    own = paged.build_tables(context, new, tables[0], free, ints([2], cuda), bs, 6)
    given = paged.StepTables(*(torch.full_like(x, -9) for x in own))
    assert paged.build_tables(context, new, tables[1], free, ints([2], cuda), bs, 6, out=given) is given
    assert torch.equal(tables[0], tables[1]) and all(torch.equal(a, b) for a, b in zip(own, given))

    x = torch.randn(6, heads + 2 * hk, dim, device=cuda).half()
    freqs = torch.randn(64, dim // 2, 2, device=cuda)
    kc, ks = make_cache(20, hk, bs, dim, "e4m3", cuda, 1)
    vc, vs = make_cache(20, hk, bs, dim, "e4m3", cuda, 2)
    copies = [kc.clone(), vc.clone(), ks.clone(), vs.clone()]
    args = (x[:, heads:heads + hk], x[:, heads + hk:], own.slots)
    q = paged.append_kv8(*args, kc, vc, ks, vs, q=x[:, :heads], freqs=freqs, positions=own.positions)
    q_out = torch.empty(6, heads, dim, dtype=torch.float16, device=cuda)
    got = paged.append_kv8(*args, *copies, q=x[:, :heads], freqs=freqs, positions=own.positions, q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr() and torch.equal(q, q_out)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((kc, vc, ks, vs), copies))

    attend = lambda out=None: paged.attend_kv8(q, kc, vc, ks, vs, tables[0], own.seq_lens, own.query_starts, 3, out=out)  # noqa: E731
    out = torch.full_like(q, math.nan)
    assert attend(out).data_ptr() == out.data_ptr() and torch.equal(out, attend())

    logits, u = torch.randn(7, 3001, device=cuda), torch.rand(7, device=cuda)
    t, lp = sampling.sample(logits, u, top_p=torch.full((7,), 0.7, device=cuda))
    tokens, logprobs = torch.empty_like(t), torch.empty_like(lp)
    a, b = sampling.sample(logits, u, top_p=torch.full((7,), 0.7, device=cuda), tokens=tokens, logprobs=logprobs)
    assert a.data_ptr() == tokens.data_ptr() and b.data_ptr() == logprobs.data_ptr() and torch.equal(t, tokens) and torch.equal(lp, logprobs)
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("new", [1, 40])
def test_overlapping_launches(cuda, new):
    """Steps of several layers with each launch beginning before the one ahead of it has ended: the same bits, eagerly and from a graph."""
    bs, heads, hk, dim, requests, layers = 16, 8, 2, 128, 5, 4
    context = ints([0, 5, 16, 40, 300], cuda)
    free = torch.arange(100, dtype=torch.int32, device=cuda)
    x = torch.randn(layers, requests * new, heads + 2 * hk, dim, device=cuda).half()
    freqs = torch.randn(400, dim // 2, 2, device=cuda)
    first = [make_cache(130, hk, bs, dim, "int8", cuda, i) for i in range(2 * layers)]
    row = torch.full((requests, 24), -1, dtype=torch.int32, device=cuda)
    row[1, 0], row[2, 0], row[3, :3], row[4, :19] = 100, 101, ints([102, 103, 104], cuda), ints(list(range(105, 124)), cuda)
    ws = paged.attend_workspace(requests, new, heads, hk, dim, cuda)
    u = torch.rand(requests, device=cuda)
    head, lens = ints([0], cuda), ints([new] * requests, cuda)

    def step(caches, table):
        t = paged.build_tables(context, lens, table, free, head, bs, requests * new)
        a, outs = None, []
        for i in range(layers):
            (kc, ks), (vc, vs) = caches[2 * i], caches[2 * i + 1]
            k = x[i, :, heads:heads + hk]
            q = paged.append_kv8(k, x[i, :, heads + hk:], t.slots, kc, vc, ks, vs, q=x[i, :, :heads] if a is None else a, freqs=freqs,
                                 positions=t.positions)
            a = paged.attend_kv8(q, kc, vc, ks, vs, table, t.seq_lens, t.query_starts, new, workspace=ws)
            outs.append(a)
        tokens, lp = sampling.sample(a.view(requests, -1)[:, :heads * dim].float(), u, temperature=torch.full_like(u, 0.8))
        return torch.stack(outs), tokens, lp

    fresh = lambda: ([(c.clone(), s.clone()) for c, s in first], row.clone())  # noqa: E731
    want = step(*fresh())
    capi.set_pdl(True)
    try:
        for _ in range(20):
            state = fresh()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, step(*state)))
        state = fresh()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(*state)
        for _ in range(5):
            for (c, s), (c0, s0) in zip(state[0], first):
                c.copy_(c0)
                s.copy_(s0)
            state[1].copy_(row)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    finally:
        capi.set_pdl(False)
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_error_of_a_block_filled_token_by_token(cuda, kind):
    """What a block holds in the end against what went in, when its scale grows at most calls.  A code is rounded when it is written and
    again at each growth (an e4m3 code only at one that more than doubles): each time by half a step of an int8 code, or by 2^-4 of
    the value or 2^-10 of the scale where that is more."""
    bs, dim, runs = 128, 64, 8
    gen = torch.Generator(device=cuda).manual_seed(11)
    # magnitudes that grow by 2.1 to 5 at a time, then stay: the early tokens are rounded again and again
    steps = 2.1 + 2.9 * torch.rand(runs, generator=gen, device=cuda)
    size = torch.cat([torch.cumprod(steps, 0), steps.prod().expand(bs - runs)]) * 2.0 ** -10
    x = torch.randn(bs, 1, dim, generator=gen, device=cuda)
    x = (x / x.abs().amax(-1, keepdim=True) * size[:, None, None]).half()
    kc, vc = (torch.zeros(1, 1, bs, dim, dtype=torch.uint8, device=cuda).view(CODE[kind]) for _ in range(2))
    ks, vs = torch.zeros(1, 1, device=cuda), torch.zeros(1, 1, device=cuda)
    exact = x[:, 0].double()
    bound = torch.zeros(bs, dim, dtype=torch.float64, device=cuda)
    last = 0.0
    for i in range(bs):
        paged.append_kv8(x[i:i + 1], -x[i:i + 1], ints([i], cuda, torch.int64), kc, vc, ks, vs)
        s = ks[0, 0].item()
        # one rounding of what the codes are before it: the value and its error so far
        rounding = torch.full_like(bound, 0.5 * s) if kind == "int8" else torch.maximum(2.0 ** -4 * (exact.abs() + bound), torch.tensor(2.0 ** -10 * s, device=cuda))
        rounding = rounding * (1 + 2.0 ** -10)
        bound[i] = rounding[i]
        if i and s != last:
            bound[:i] += rounding[:i]
        last = s
    for c, s, w in ((kc, ks, exact), (vc, vs, -exact)):
        assert bool(((c[0, 0].double() * s[0, 0].double() - w).abs() <= bound).all())
    # the growths more than double, so the roundings of an int8 code add up to less than a step of the last scale
    if kind == "int8":
        assert bound.max().item() <= 1.002 * last
    assert capi.device_error(0) == 0
