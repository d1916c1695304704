"""Attention's schedule: how the work of many requests is cut over the CTAs.  Every call is checked against the 64-bit restatement
and against itself, since a schedule on which a CTA's warps disagree shows in some calls only."""
from __future__ import annotations

import math
import random

import pytest
import torch

from gdsllm_b200 import capi, paged
from test_paged_gpu import attend_ref, ints, make_cache

pytestmark = pytest.mark.gpu


def check_repeated(cuda, kind, heads, kv_heads, dim, bs, lens, new, times, seed):
    rng = random.Random(seed)
    blocks = [-(-n // bs) for n in lens]
    ids = list(range(sum(blocks) + 2))
    rng.shuffle(ids)
    width = max(blocks) + 1
    table = ints([[ids.pop() for _ in range(b)] + [-1] * (width - b) for b in blocks], cuda)
    kc, ks = make_cache(sum(blocks) + 2, kv_heads, bs, dim, kind, cuda, seed + 1)
    vc, vs = make_cache(sum(blocks) + 2, kv_heads, bs, dim, kind, cuda, seed + 2)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], heads, dim, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).half()
    ws = paged.attend_workspace(len(lens), max(new), heads, kv_heads, dim, cuda)
    call = lambda: paged.attend_kv8(q, kc, vc, ks, vs, table, ints(lens, cuda), ints(starts, cuda), max(new), workspace=ws)  # noqa: E731
    first = call()
    want, bound = attend_ref(q, kc, vc, ks, vs, table, lens, starts, 1 / math.sqrt(dim), 2.0 ** -11)
    assert bool(((first.double() - want).abs() <= bound).all())
    differ = torch.zeros((), dtype=torch.int64, device=cuda)
    for _ in range(times):
        differ += (call() != first).sum()
    assert differ.item() == 0
    assert capi.device_error(0) == 0


# From 2 requests on, the thread that finds a CTA's first request writes where it begins while other warps may still add up the sums.
@pytest.mark.parametrize("requests", [2, 3, 31, 513, 700])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (16, 1, 256), (10, 2, 64)])
def test_tile_schedule(cuda, requests, heads, kv_heads, dim):
    rng = random.Random(requests)
    new = [40] + [rng.choice([0, 1, 5, 17, 40]) for _ in range(requests - 1)]
    lens = [n + rng.choice([0, 1, 63, 130, 300]) for n in new]
    check_repeated(cuda, "e4m3", heads, kv_heads, dim, 16, [max(n, 1) for n in lens], new, 200, requests + dim)


@pytest.mark.parametrize("requests", [2, 129, 300, 1000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (10, 1, 256), (24, 1, 64)])
def test_stream_schedule(cuda, requests, heads, kv_heads, dim):
    rng = random.Random(requests)
    lens = [rng.choice([1, 15, 64, 130, 300]) for _ in range(requests)]
    check_repeated(cuda, "int8", heads, kv_heads, dim, 16, lens, [1] + [rng.choice([0, 1]) for _ in range(requests - 1)], 200, requests + dim)


def test_prompts_beside_single_tokens(cuda):
    """One prompt chunk among decoding requests: all of them take the kernel that its rows ask for."""
    rng = random.Random(6)
    new = [1] * 47 + [600] + [1] * 16
    check_repeated(cuda, "e4m3", 16, 2, 128, 64, [n + rng.randrange(2000) for n in new], new, 50, 6)
