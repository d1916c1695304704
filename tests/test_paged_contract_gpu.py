"""What the batched-serving calls promise beside their formulas: padded steps, given outputs, hints, launches that overlap."""
from __future__ import annotations

import math

import pytest
import torch

from gdsllm_b200 import capi, paged
from test_paged_gpu import attend_ref, ints, make_cache

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
