"""Sampling against a plain restatement with whole-number weights."""
from __future__ import annotations

import math

import pytest
import torch

from gdsllm_b200 import sampling

pytestmark = pytest.mark.gpu


def sample_ref(row, u, temp, k, p, mp):
    """One row: (token, logprob in 64 bits).  The weights are whole by definition (the exponential is the 32-bit one)."""
    x = torch.where(torch.isnan(row.float()), -math.inf, row.float())
    v = x.numel()
    greedy = not temp > 0
    inv = 1.0 if greedy else torch.reciprocal(torch.tensor(temp, dtype=torch.float32, device=x.device))
    top = x.max()
    if top == -math.inf:
        return -1, -math.inf
    e = torch.where(x == top, 1.0, torch.exp((x - top) * inv))
    e = torch.where(x == -math.inf, 0.0, e)
    w = torch.floor(e.double() * 2.0 ** 31)
    order = torch.sort(x, descending=True, stable=True).indices
    k = 1 if greedy else (k if 0 < k < v else v)
    order = order[:k]
    total = w[order].sum()
    before = torch.cumsum(w[order], 0) - w[order]
    keep = (before < torch.tensor(p, dtype=torch.float32).double().item() * total) & (e[order] >= mp)
    keep[0] = True
    chosen = torch.sort(order[keep]).values
    run = torch.cumsum(w[chosen], 0)
    target = torch.clamp(torch.floor(u.double() * run[-1]), max=run[-1] - 1)
    i = chosen[torch.searchsorted(run, target.reshape(1), right=True)[0]]
    return i.item(), torch.log(w[i] / run[-1]).item()


def check(logits, u, temp=None, k=None, p=None, mp=None):
    dev = logits.device
    b = logits.shape[0]

    def col(v, dtype=torch.float32):
        return None if v is None else torch.tensor(v, dtype=dtype, device=dev)
    tokens, lp = sampling.sample(logits, u, temperature=col(temp), top_k=col(k, torch.int32), top_p=col(p), min_p=col(mp))
    for i in range(b):
        def f32(v, default):
            return default if v is None else torch.tensor(v[i], dtype=torch.float32).item()
        want, wlp = sample_ref(logits[i], u[i], f32(temp, 1.0), 0 if k is None else k[i], f32(p, 1.0), f32(mp, 0.0))
        assert tokens[i].item() == want, (i, tokens[i].item(), want)
        # a quotient rounded to 32 bits, then logf: 2^-23 of the quotient and a unit in the last place
        assert lp[i].item() == wlp or abs(lp[i].item() - wlp) <= 2.0 ** -22 * (1 + abs(wlp))
    return tokens, lp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 32000, 50001, 131072, 300007])
def test_sample(cuda, dtype, vocab):
    b = 24
    gen = torch.Generator(device=cuda).manual_seed(vocab)
    x = 2.5 * torch.randn(b, vocab, generator=gen, device=cuda)
    x[:, :: max(1, vocab // 9)] += 5
    x = x.to(dtype)
    u = torch.rand(b, generator=gen, device=cuda)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    check(x, u)
    ks = [0, 1, 2, 5, 40, 1000, vocab, vocab + 7] * 3
    ps = [1.0, 0.9, 0.5, 0.0, 0.999, 1e-6, 0.95] * 4
    ms = [0.0, 0.05, 0.5, 1.0, 0.0] * 5
    ts = [1.0, 0.7, 0.0, 1.6, 0.3, 100.0, 1e-4, 0.9] * 3
    check(x, u, temp=ts[:b], k=ks[:b], p=ps[:b], mp=ms[:b])
    check(x, u, p=ps[:b])
    check(x, u, k=ks[:b])
    check(x, u, temp=ts[:b], mp=ms[:b])


def test_ties(cuda):
    """Equal logits at every cut: the lowest indices stay."""
    b, v = 40, 5000
    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randint(0, 4, (b, v), generator=gen, device=cuda).half()
    u = torch.rand(b, generator=gen, device=cuda)
    check(x, u, k=[1 + 61 * i for i in range(b)])
    check(x, u, p=[(i + 1) / b for i in range(b)])
    check(x, u, k=[3 + 97 * i for i in range(b)], p=[(i + 0.5) / b for i in range(b)])
    same = torch.zeros(b, v, device=cuda)
    same[:, 100:200] = -0.0
    check(same, u, k=[0, 1, 150, 4999] * 10, p=[1.0, 0.5, 0.037] * 13 + [0.2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_infinities_and_nan(cuda, dtype):
    b, v = 8, 3001
    gen = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(b, v, generator=gen, device=cuda).to(dtype)
    x[0] = -math.inf
    x[1, 5:] = -math.inf
    x[2, 77] = math.nan
    x[3, :] = math.nan
    x[4, [9, 2000]] = math.inf
    x[5, ::2] = math.nan
    x[6, :] = torch.finfo(dtype).min
    x[7, 1:] = torch.finfo(dtype).min
    u = torch.rand(b, generator=gen, device=cuda)
    for kw in ({}, {"k": [7] * b}, {"p": [0.6] * b}, {"temp": [0.0] * b}, {"k": [0, 3000, 50, 2, 1, 9, 3, 2], "p": [0.9] * b, "mp": [0.1] * b}):
        tokens, _ = check(x, u, **kw)
        assert tokens[0] == -1 and tokens[3] == -1 and 0 <= tokens[1] < 5 and tokens[4] in (9, 2000) and tokens[5] % 2 == 1


def test_strided_rows_and_repeatability(cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    x = torch.randn(33, 4099, generator=gen, device=cuda).half()
    u = torch.rand(33, generator=gen, device=cuda)
    part = x[:, 1:4001]  # odd stride, rows that start off alignment
    a, la = check(part, u, p=[0.8] * 33)
    for _ in range(3):
        c, lc = sampling.sample(part, u, top_p=torch.full((33,), 0.8, device=cuda))
        assert torch.equal(a, c) and torch.equal(la, lc)


def test_frequencies(cuda):
    """20000 draws from one distribution: every token's count within 6 standard deviations of its probability."""
    n, v = 20000, 40
    gen = torch.Generator(device=cuda).manual_seed(7)
    row = 1.5 * torch.randn(v, generator=gen, device=cuda)
    u = torch.rand(n, generator=gen, device=cuda)
    tokens, _ = sampling.sample(row.repeat(n, 1), u)
    p = torch.softmax(row.double(), 0)
    count = torch.bincount(tokens, minlength=v).double()
    assert bool(((count - n * p).abs() <= 6 * torch.sqrt(n * p * (1 - p)) + 1).all())


@pytest.mark.parametrize("vocab", [131072, 200000])
def test_flat_rows_of_a_large_vocabulary(cuda, vocab):
    """More than 2^16 logits of one value in a row that few CTAs share: sums of 2^48 and more."""
    b = 300
    x = torch.full((b, vocab), -3.0, dtype=torch.float16, device=cuda)
    x[0] = 0.0
    x[1::2, 7] = 0.0
    u = torch.rand(b, generator=torch.Generator(device=cuda).manual_seed(5), device=cuda)
    tokens, lp = sampling.sample(x, u, top_p=torch.full((b,), 0.5, device=cuda))
    for i in (0, 1, 2, 3, 150, 299):
        want, wlp = sample_ref(x[i], u[i], 1.0, 0, 0.5, 0.0)
        assert tokens[i].item() == want
        assert abs(lp[i].item() - wlp) <= 2.0 ** -22 * (1 + abs(wlp))
