"""Attention over the 8-bit cache at long lengths, with bounds tight enough that a lost or doubled tile of 32 tokens shows, and at
weights far below the largest.  The inputs are made on the CPU; there the reference is given such mistakes (marked tests run on the GPU)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from gdsllm_b200 import capi, paged

CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
BS, TILE = 64, 32


class Case:
    """One request of n tokens, the last ``new`` of them queries; K and V codes by token with a scale per block, as written and as read."""

    def __init__(self, kind, heads, dim, n, new, k, v, q, ks, vs, scale):
        self.kind, self.heads, self.dim, self.n, self.new, self.k, self.v, self.q, self.ks, self.vs, self.scale = kind, heads, dim, n, new, k, v, q, ks, vs, scale

    def parts(self, dev):
        """(x, vq, p, o, sums) in 64 bits for rows [new * heads]: x = exp(s - max) * vs, p the softmax."""
        at = torch.arange(self.n, device=dev) // BS
        k = self.k.to(dev).double() * self.ks.to(dev).double()[at, None]
        s = self.q.to(dev).double().reshape(-1, self.dim) @ k.T * self.scale
        row = torch.arange(self.new * self.heads, device=dev) // self.heads
        s = s.masked_fill(torch.arange(self.n, device=dev)[None] > (self.n - self.new + row)[:, None], -math.inf)
        e = torch.exp(s - s.amax(1, keepdim=True))
        reach = (self.q.to(dev).double().abs().reshape(-1, self.dim) @ k.abs().T * abs(self.scale)).amax(1, keepdim=True)
        return e, e * self.vs.to(dev).double()[at], self.v.to(dev).double(), reach

    def exact(self, dev, independent):
        """(o, bound).  What a weight x_j = e_j vs_j loses by 16 bits: 2^-11 of itself, or 2^-32 of the largest where that is more (but not
        more than itself).  Added up as they are, or, where the weights differ and so are rounded independently, as 8 standard
        deviations.  The fp32 sums: 2^-16 of sum p|v|; the scores' sums: 2^-18 of sum |q||k|; the output: 2^-11 of itself (bf16: 2^-8), 2^-24."""
        eps = 2.0 ** -11 if self.q.dtype == torch.float16 else 2.0 ** -8
        e, x, vq, reach = self.parts(dev)
        den, most = e.sum(1, keepdim=True), x.amax(1, keepdim=True)
        o = x @ vq / den
        small = torch.minimum(x, 2.0 ** -32 * most)
        if independent:
            lost = 8 * 2.0 ** -11 * torch.sqrt(x ** 2 @ vq ** 2) + small @ vq.abs()
        else:
            lost = torch.maximum(2.0 ** -11 * x, small) @ vq.abs()
        bound = (lost + (2.0 ** -16 + 2.0 ** -18 * reach) * (x @ vq.abs())) / den + o.abs() * eps + 2.0 ** -24
        return o, bound

    def run(self, dev, requests=1):
        """The operator on a shuffled pool, for ``requests`` alike that share its blocks: [requests, rows, dim]."""
        blocks = -(-self.n // BS)
        order = list(range(blocks + 1))
        random.Random(self.n).shuffle(order)
        order = torch.tensor(order[:blocks], device=dev)
        caches, scales = [], []
        for codes, s in ((self.k, self.ks), (self.v, self.vs)):
            c = torch.full(((blocks + 1) * BS, self.dim), 0x7F if self.kind == "e4m3" else 0x80, dtype=torch.uint8, device=dev)
            at = torch.arange(self.n, device=dev)
            c[order[at // BS] * BS + at % BS] = codes.to(CODE[self.kind]).view(torch.uint8).to(dev)
            caches.append(c.view(blocks + 1, 1, BS, self.dim).view(CODE[self.kind]))
            t = torch.zeros(blocks + 1, 1, device=dev)
            t[order, 0] = s.to(dev)
            scales.append(t)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        q = self.q.to(dev).repeat(requests, 1, 1)
        starts = [self.new * r for r in range(requests + 1)]
        return paged.attend_kv8(q, *caches, *scales, order.int()[None].repeat(requests, 1), i32([self.n] * requests), i32(starts), self.new,
                                softmax_scale=self.scale).view(requests, -1, self.dim)

    def check(self, dev, independent, requests=1):
        got = self.run(dev, requests).double()
        o, bound = self.exact(dev, independent)
        err = (got - o).abs()
        assert bool((err <= bound).all()), f"worst error / bound {(err / bound).max().item()}"
        assert capi.device_error(0) == 0


def flat_case(kind, heads, dim, n, new, seed=0):
    """A softmax that no token dominates, and values whose signs differ from tile to tile of 32 tokens."""
    gen = torch.Generator().manual_seed(seed + n + dim)
    top = TOP[kind]
    k = (torch.randn(n, dim, generator=gen) * top / 4).clamp(-top, top)
    k = k.round() if kind == "int8" else k.to(CODE[kind]).float()
    sign = torch.randint(0, 2, (-(-n // TILE), dim), generator=gen).repeat_interleave(TILE, 0)[:n] * 2 - 1
    v = sign * torch.randint(10, 15, (n, dim), generator=gen) * 8.0  # 80 to 112: codes of either kind
    blocks = -(-n // BS)
    ks = (4 / top) * (1 + 0.2 * torch.rand(blocks, generator=gen))
    vs = 0.01 * (1 + 0.1 * torch.rand(blocks, generator=gen))
    q = (0.3 * torch.randn(new, heads, dim, generator=gen)).half()
    return Case(kind, heads, dim, n, new, k, v, q, ks, vs, 1 / math.sqrt(dim))


def sink_case(kind, heads, dim, n, new, bits):
    """The first token's weight is 2^bits times each other's; its value is 0, the others' is not."""
    k, v = torch.zeros(n, dim), torch.full((n, dim), 96.0)
    k[0], v[0] = 64.0, 0.0
    q = torch.full((new, heads, dim), 0.5).half()
    blocks = -(-n // BS)
    ks = torch.full((blocks,), 0.015625)
    return Case(kind, heads, dim, n, new, k, v, q, ks, torch.full((blocks,), 0.01), bits * math.log(2.0) / (64 * 0.015625 * 0.5 * dim))


SHAPES = [("int8", 2, 128, 70001, 1), ("e4m3", 8, 64, 70001, 3), ("e4m3", 2, 256, 40003, 2),   # up to 32 rows
          ("e4m3", 8, 128, 70001, 40), ("int8", 3, 64, 30007, 17), ("int8", 16, 256, 40003, 9)]  # more


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,dim,n,new", SHAPES)
def test_long_and_flat(cuda, kind, heads, dim, n, new):
    flat_case(kind, heads, dim, n, new).check(cuda, independent=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,dim,n,new", SHAPES[3:])
def test_long_and_flat_for_many_requests(cuda, kind, heads, dim, n, new):
    """More requests than two thirds of the CTAs: each takes tens of thousands of tokens of a request and leaves it to the next."""
    flat_case(kind, heads, dim, n, new).check(cuda, independent=True, requests=101)


@pytest.mark.parametrize("kind,heads,dim,n,new", [s[:4] + (1,) for s in SHAPES])
def test_the_bound_shows_a_lost_or_doubled_tile(kind, heads, dim, n, new):
    """Every tile of 32 tokens, left out of the reference or counted twice, takes some output further than twice the bound."""
    case = flat_case(kind, heads, dim, n, new)
    e, x, vq, _ = case.parts("cpu")
    o, bound = case.exact("cpu", independent=True)
    tiles = -(-n // TILE)
    pad = tiles * TILE - n
    e = torch.nn.functional.pad(e, (0, pad)).view(-1, tiles, TILE)
    x = torch.nn.functional.pad(x, (0, pad)).view(-1, tiles, TILE)
    num = torch.einsum("rtj,tjd->rtd", x, torch.nn.functional.pad(vq, (0, 0, 0, pad)).view(tiles, TILE, -1))
    den = e.sum(2, keepdim=True)
    whole = n // TILE  # the last tile may hold a single token
    for times in (-1, 1):
        wrong = (num.sum(1, keepdim=True) + times * num) / (den.sum(1, keepdim=True) + times * den)
        worst = ((wrong - o[:, None]).abs() / bound[:, None]).amax((0, 2))[:whole]
        assert worst.min().item() > 2, worst.min().item()


# 2^-25.2 of the largest is below fp16's smallest number, 2^-24.4 a little above it.  As many requests as keep a CTA at one of them, so
# that its weights share a reference point.
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [10.3, 20.5, 24.4, 25.2, 28.0])
@pytest.mark.parametrize("kind,heads,dim,n,new", [("int8", 4, 128, 131072, 1), ("e4m3", 1, 64, 131071, 3), ("e4m3", 4, 256, 100003, 1),
                                                  ("e4m3", 8, 128, 131072, 5), ("int8", 33, 64, 131072, 1), ("int8", 20, 256, 100003, 1)])
def test_many_small_weights_beside_a_large_one(cuda, kind, heads, dim, n, new, bits):
    sink_case(kind, heads, dim, n, new, bits).check(cuda, independent=False, requests=444)


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [2.0 ** -12, 2.0 ** -17, 2.0 ** -22])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind,heads,dim,n,new", [("int8", 4, 64, 50, 1), ("e4m3", 2, 128, 50, 8), ("int8", 2, 256, 50, 8),
                                                  ("e4m3", 1, 64, 90, 40), ("int8", 2, 128, 90, 40), ("e4m3", 2, 256, 90, 40)])
def test_small_query_elements_beside_a_large_one(cuda, kind, heads, dim, n, new, dtype, ratio):
    """The query's largest element meets keys of zero: the scores come from elements far smaller."""
    gen = torch.Generator().manual_seed(dim + new)
    top = TOP[kind]
    k = (torch.randn(n, dim, generator=gen) * top / 4).clamp(-top, top)
    k = k.round() if kind == "int8" else k.to(CODE[kind]).float()
    k[:, 5] = 0
    q = torch.randn(new, heads, dim, generator=gen) * ratio
    q[:, :, 5] = 1.0
    blocks = -(-n // BS)
    Case(kind, heads, dim, n, new, k, torch.randint(-14, 15, (n, dim), generator=gen) * 8.0, (q * 50000).to(dtype), torch.full((blocks,), 4 / top),
         torch.full((blocks,), 0.01), 4 / (50000 * ratio * math.sqrt(dim))).check(cuda, independent=False)


@pytest.mark.gpu
@pytest.mark.parametrize("log_scale", [-96, 60, 99, 105, 119])
@pytest.mark.parametrize("kind,heads,dim,n,new", [("int8", 4, 128, 300, 1), ("e4m3", 8, 64, 300, 3), ("e4m3", 4, 256, 300, 9), ("int8", 8, 128, 300, 40)])
def test_value_scales_over_bf16s_range(cuda, kind, heads, dim, n, new, log_scale):
    """Values far outside fp16's range; the largest are 2^126."""
    case = flat_case(kind, heads, dim, n, new)
    case.q, case.vs = case.q.bfloat16(), case.vs * 2.0 ** (log_scale - math.log2(case.vs[0].item()))
    case.check(cuda, independent=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 40])
def test_large_bf16_values_written_and_read(cuda, kind, new):
    """Written by the cache write, read by attention: one token's value comes back."""
    dim, n = 64, 40
    caches = [torch.zeros(1, 1, BS, dim, dtype=torch.uint8, device=cuda).view(CODE[kind]) for _ in range(2)]
    scales = [torch.zeros(1, 1, device=cuda) for _ in range(2)]
    v = torch.full((n, 1, dim), 2.0 ** 125, dtype=torch.bfloat16, device=cuda)
    i32 = lambda *t: torch.tensor(t, dtype=torch.int32, device=cuda)  # noqa: E731
    paged.append_kv8(torch.zeros_like(v), v, torch.arange(n, device=cuda), *caches, *scales)
    q = torch.ones(new, 1, dim, dtype=torch.bfloat16, device=cuda)
    got = paged.attend_kv8(q, *caches, *scales, i32(0)[None], i32(n), i32(0, new), new)
    # the code is top itself; the scale's rounding, the weights' and bf16's
    assert bool(((got.double() / 2.0 ** 125 - 1).abs() <= 2.0 ** -8 + 2.0 ** -10).all())
