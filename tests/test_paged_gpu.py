"""The paged 8-bit cache: step tables, cache write and attention against
plain 64-bit restatements, at the sizes, masks and layouts where they can go
wrong.  Tolerances are derived beside each check from the roundings that the
definition has."""
from __future__ import annotations

import math
import random

import pytest
import torch

from gdsllm_b200 import capi, paged

pytestmark = pytest.mark.gpu

CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
HALF = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(1234)


def ints(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


# ---- step tables ------------------------------------------------------------------

def tables_ref(context, new, table, free, head, bs, tokens):
    table = [list(r) for r in table]
    starts, positions, slots = [0], [], []
    for r, (c, n) in enumerate(zip(context, new)):
        for j in range(-(-c // bs), -(-(c + n) // bs)):
            table[r][j] = free[head]
            head += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r][p // bs] * bs + p % bs)
        starts.append(starts[-1] + n)
    pad = tokens - len(slots)
    return table, starts, positions + [0] * pad, slots + [-1] * pad, head


@pytest.mark.parametrize("requests,bs,longest,spare", [(1, 16, 1, 0), (1, 64, 1000, 5), (7, 16, 40, 3), (64, 64, 1, 0),
                                                       (257, 128, 300, 17), (1025, 32, 90, 0), (3000, 16, 9, 1)])
def test_tables(cuda, requests, bs, longest, spare):
    rng = random.Random(requests * 131 + bs)
    context = [rng.choice([0, 1, bs - 1, bs, bs + 1, rng.randrange(6 * bs)]) for _ in range(requests)]
    new = [rng.choice([0, 1, longest, rng.randint(0, longest)]) for _ in range(requests)]
    width = max(-(-(c + n) // bs) for c, n in zip(context, new)) + 2
    ids = list(range(requests * width * 2))
    rng.shuffle(ids)
    table = [[-7] * width for _ in range(requests)]
    for r, c in enumerate(context):
        for j in range(-(-c // bs)):
            table[r][j] = ids.pop()
    total = sum(new) + spare
    want = tables_ref(context, new, table, ids, 3, bs, total)
    t = ints(table, cuda)
    got = paged.build_tables(ints(context, cuda), ints(new, cuda), t, ints(ids, cuda), ints([3], cuda), bs, total)
    assert t.tolist() == want[0]
    assert got.query_starts.tolist() == want[1]
    assert got.positions.tolist() == want[2]
    assert got.slots.tolist() == want[3]
    assert got.free_head.tolist() == [want[4]]
    assert got.seq_lens.tolist() == [c + n for c, n in zip(context, new)]
    assert capi.device_error(0) == 0


def test_tables_short_queue_and_row(cuda):
    """Too few free blocks, a row that is too short, a negative length and too few token places: -1 and the error bit."""
    bs = 16
    t = ints([[-1, -1], [-1, -1]], cuda)
    got = paged.build_tables(ints([0, 0], cuda), ints([20, 20], cuda), t, ints([5, 9, 11], cuda), ints([0], cuda), bs, 40)
    assert t.tolist() == [[5, 9], [11, -1]]
    assert got.slots[:20].tolist() == [5 * bs + i for i in range(16)] + [9 * bs + i for i in range(4)]
    assert got.slots[20:36].tolist() == [11 * bs + i for i in range(16)] and got.slots[36:].tolist() == [-1] * 4
    assert capi.device_error(0) == 4
    t = ints([[-1]], cuda)
    got = paged.build_tables(ints([0], cuda), ints([17], cuda), t, ints([5, 9, 11], cuda), ints([0], cuda), bs, 17)
    assert t.tolist() == [[5]] and got.slots.tolist() == [5 * bs + i for i in range(16)] + [-1]
    assert capi.device_error(0) == 4
    got = paged.build_tables(ints([0], cuda), ints([3], cuda), t, ints([5], cuda), ints([0], cuda), bs, 2)
    assert got.slots.tolist() == [80, 81]
    assert capi.device_error(0) == 4
    paged.build_tables(ints([-1], cuda), ints([3], cuda), t, ints([5], cuda), ints([0], cuda), bs, 3)
    assert capi.device_error(0) == 4
    assert capi.device_error(0) == 0


def test_tables_lengths_near_the_largest_int(cuda):
    """Lengths that no table holds: reported, the rows' own neighbours untouched, the sums stop at the largest int."""
    big, bs = 2 ** 31 - 1, 16
    table = torch.full((3, 4), -7, dtype=torch.int32, device=cuda)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    t = paged.build_tables(i32(big, 0, 3), i32(5, 2, 2), table, i32(4, 5, 6, 7), i32(0), bs, 9)
    assert capi.device_error(0) == 4
    assert table[0].tolist() == [-7] * 4 and table[1].tolist()[1:] == [-7] * 3 and table[2].tolist() == [-7] * 4
    assert t.query_starts.tolist() == [0, 5, 7, 9] and t.slots[:5].tolist() == [-1] * 5
    assert t.slots[5:7].tolist() == [table[1, 0].item() * bs, table[1, 0].item() * bs + 1]
    t = paged.build_tables(i32(0, 0, 0), i32(big, big, big), table, i32(4, 5, 6, 7), i32(0), bs, 20)
    assert capi.device_error(0) == 4
    assert table[0].tolist() == [4, 5, 6, 7] and t.slots.tolist() == [4 * bs + i for i in range(16)] + [5 * bs + i for i in range(4)]
    assert t.query_starts.tolist()[3] == big
    assert capi.device_error(0) == 0



# ---- cache write ------------------------------------------------------------------

def append_ref(x, slots, cache, scale, kind):
    """Block by block in 64 bits from 32-bit inputs: (codes before rounding, scales); slots < 0 are skipped."""
    bs = cache.shape[2]
    cache, scale = cache.double(), scale.double()
    i, n = 0, len(slots)
    while i < n:
        if slots[i] < 0:
            i += 1
            continue
        j = i
        while j < n and slots[j] >= 0 and slots[j] // bs == slots[i] // bs:
            j += 1
        page, begin = slots[i] // bs, slots[i] % bs
        need = x[i:j].double().abs().amax((0, 2)) / TOP[kind]
        base = scale[page] if begin else torch.zeros_like(need)
        new = torch.where(need <= base, base, torch.maximum(need, 2 * base))
        cache[page, :, :begin] *= torch.where(new > 0, base / new, torch.ones_like(new))[:, None, None]
        inv = torch.where(new > 0, 1 / new, torch.zeros_like(new))
        cache[page][:, [s % bs for s in slots[i:j]]] = (x[i:j].double() * inv[None, :, None]).transpose(0, 1)
        scale[page] = new
        i = j
    return cache, scale


def rotated(x, freqs, positions):
    z = torch.view_as_complex(freqs.double())[positions][:, None]
    xc = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
    return torch.view_as_real(xc * z).flatten(-2)


def angles(dim, n, dev):
    a = torch.outer(torch.arange(n, device=dev).float(), 10000.0 ** (-torch.arange(0, dim, 2, device=dev).float() / dim))
    return torch.stack([a.cos(), a.sin()], -1).contiguous()


def check_codes(got, want, kind, what):
    """One rounding of the exact quotient, in which 1/scale and the product carry 2^-22 relative at most: int8 within 0.5 + 2^-14
    of a step; e4m3 within half a step of its 3-bit mantissa (2^-4 relative, 2^-10 under the normals) and that."""
    err = (got.double() - want).abs()
    bound = torch.full_like(want, 0.5 + 2.0 ** -14) if kind == "int8" else want.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10
    assert bool((err <= bound).all()), f"{what}: worst excess {(err - bound).max().item()}"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,bs", [("f16", 8, 8, 64, 16), ("bf16", 16, 2, 128, 32), ("f16", 12, 4, 128, 64),
                                                         ("bf16", 8, 1, 256, 128), ("f16", 64, 8, 128, 64), ("f16", 6, 3, 256, 16)])
@pytest.mark.parametrize("rope", [False, True])
def test_append(cuda, kind, dtype, heads, kv_heads, dim, bs, rope):
    rng = random.Random(heads * 7 + bs + rope)
    gen = torch.Generator(device=cuda).manual_seed(heads + bs)
    runs = [(0, 1), (1, 1), (bs - 1, 1), (bs - 1, 2), (3, bs), (0, bs), (5, 3 * bs + 1), (0, 0), (2 * bs, 1)]
    context, new = [c for c, _ in runs], [n for _, n in runs]
    blocks = [-(-(c + n) // bs) for c, n in runs]
    pool = sum(blocks) + 4
    ids = list(range(pool))
    rng.shuffle(ids)
    slots, positions = [], []
    for (c, n), b in zip(runs, blocks):
        mine = [ids.pop() for _ in range(b)]
        positions += range(c, c + n)
        slots += [mine[p // bs] * bs + p % bs for p in range(c, c + n)]
    slots.insert(3, -1)  # a padded place inside the batch
    positions.insert(3, 0)
    slots += [-1, -1]
    positions += [0, 0]
    t = len(slots)
    qkv = torch.randn(t, heads + 2 * kv_heads, dim, generator=gen, device=cuda).to(HALF[dtype])
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    v[-4] *= 20  # a token that makes its block's scale grow
    k_cache = (torch.randn(pool, kv_heads, bs, dim, generator=gen, device=cuda) * TOP[kind] / 4).clamp(-TOP[kind], TOP[kind]).to(CODE[kind])
    v_cache = k_cache.flip(0).contiguous() if kind == "int8" else k_cache.view(torch.uint8).flip(0).contiguous().view(CODE[kind])
    # scales that suffice, that are a little too small and that are far too small
    k_scale = (0.2 + 8 * torch.rand(pool, kv_heads, generator=gen, device=cuda)) / TOP[kind]
    v_scale = (0.2 + 8 * torch.rand(pool, kv_heads, generator=gen, device=cuda)) / TOP[kind]
    v_scale[::3] *= 2.0 ** -20
    freqs = angles(dim, max(positions) + 1, cuda) if rope else None
    pos = ints(positions, cuda, torch.int64)
    kx = rotated(k, freqs, pos).to(k.dtype) if rope else k
    wk, wks = append_ref(kx, slots, k_cache, k_scale, kind)
    wv, wvs = append_ref(v, slots, v_cache, v_scale, kind)
    got = paged.append_kv8(k, v, ints(slots, cuda, torch.int64), k_cache, v_cache, k_scale, v_scale, q=q if rope else None,
                           freqs=freqs, positions=pos)
    # scales: the division by 127 or 448 and, when rotated, one unit in the last place of the rounded key (2^-7 in bf16)
    one_ulp = (2.0 ** -10 if dtype == "f16" else 2.0 ** -7) if rope else 0.0
    for name, s, w, slack in (("k", k_scale, wks, one_ulp), ("v", v_scale, wvs, 0.0)):
        assert bool(((s.double() - w).abs() <= w * (2.0 ** -22 + slack)).all()), name
    if not rope:
        check_codes(k_cache, wk, kind, "k")
        # an unmoved block keeps its bits
        untouched = torch.ones(pool, dtype=torch.bool, device=cuda)
        untouched[[s // bs for s in slots if s >= 0]] = False
        assert torch.equal(k_cache[untouched].double() if kind == "int8" else k_cache.view(torch.uint8)[untouched].view(CODE[kind]).double(), wk[untouched])
    else:
        # the value: half a step of the code, and a unit in the last place of the rounded key
        value = k_cache.double() * k_scale.double()[:, :, None, None]
        exact = wk * wks[:, :, None, None]
        step = wks[:, :, None, None] * (1.01 + 2 * TOP[kind] * one_ulp if kind == "int8" else 2.0 ** -9) + exact.abs() * (one_ulp if kind == "int8" else 2.0 ** -3.9 + one_ulp)
        assert bool(((value - exact).abs() <= step).all())
        want = rotated(q, freqs, pos)
        ulp = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
        size = torch.view_as_complex(q.double().reshape(*q.shape[:-1], -1, 2).contiguous()).abs().repeat_interleave(2, -1)
        assert bool(((got.double() - want).abs() <= want.abs() * ulp + size * 2.0 ** -22 + 2.0 ** -24).all())
    check_codes(v_cache, wv, kind, "v")
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_token_by_token(cuda, kind):
    """A block filled one token at a time, each larger than the last: every call is one step of the definition on what the block
    held; and int8 ends within 1 step of what went in."""
    bs, dim = 16, 64
    x = (torch.randn(bs, 1, dim, device=cuda) * (1.3 ** torch.arange(bs, device=cuda))[:, None, None]).half()
    kc, vc = (torch.zeros(2, 1, bs, dim, dtype=torch.uint8, device=cuda).view(CODE[kind]) for _ in range(2))
    ks, vs = torch.full((2, 1), math.nan, device=cuda), torch.full((2, 1), math.nan, device=cuda)
    for i in range(bs):
        want = [append_ref(s * x[i:i + 1], [bs + i], c, sc, kind) for s, c, sc in ((1, kc, ks), (-1, vc, vs))]
        paged.append_kv8(x[i:i + 1], -x[i:i + 1], ints([bs + i], cuda, torch.int64), kc, vc, ks, vs)
        for (w, ws), c, s in zip(want, (kc, vc), (ks, vs)):
            check_codes(c, w, kind, f"token {i}")
            assert abs(s[1, 0].item() - ws[1, 0].item()) <= ws[1, 0].item() * 2.0 ** -22
    for c, s, w in ((kc, ks, x), (vc, vs, -x)):
        w = w[:, 0].double()
        if kind == "int8":
            assert bool(((c[1, 0].double() * s[1, 0].double() - w).abs() <= s[1, 0].double()).all())
        assert s[1, 0] <= 2 * w.abs().max() / TOP[kind]
    assert bool(torch.isnan(ks[0]).all()), "the other block is not touched"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_zeros_and_non_finite(cuda, kind):
    bs, dim = 16, 64
    kc, vc = (torch.zeros(3, 2, bs, dim, dtype=torch.uint8, device=cuda).view(CODE[kind]) for _ in range(2))
    ks, vs = torch.ones(3, 2, device=cuda), torch.ones(3, 2, device=cuda)
    k = torch.zeros(3, 2, dim, device=cuda).half()
    v = torch.ones(3, 2, dim, device=cuda).half()
    k[1, 0, 5] = math.inf
    v[2, 1, 7] = math.nan
    paged.append_kv8(k, v, ints([0, bs, 2 * bs], cuda, torch.int64), kc, vc, ks, vs)
    assert ks[0].tolist() == [0, 0] and bool(torch.isnan(ks[1, 0])) and ks[1, 1] == 0
    assert bool(torch.isnan(vs[2, 1])) and abs(vs[2, 0].item() - 1 / TOP[kind]) < 1e-9
    assert bool((kc.view(torch.uint8) == 0).all()) and bool((vc.view(torch.uint8)[2, 1] == 0).all())
    # the block stays marked while it fills, and is clean when begun again
    one = torch.ones(1, 2, dim, device=cuda).half()
    paged.append_kv8(one, one, ints([bs + 1], cuda, torch.int64), kc, vc, ks, vs)
    assert bool(torch.isnan(ks[1, 0])) and bool(torch.isfinite(ks[1, 1]))
    paged.append_kv8(one, one, ints([bs], cuda, torch.int64), kc, vc, ks, vs)
    assert bool(torch.isfinite(ks).all())
    assert capi.device_error(0) == 0


def test_append_bad_slot_and_position(cuda):
    bs, dim = 16, 64
    kc, vc = (torch.zeros(2, 1, bs, dim, dtype=torch.int8, device=cuda) for _ in range(2))
    ks, vs = torch.zeros(2, 1, device=cuda), torch.zeros(2, 1, device=cuda)
    x = torch.ones(1, 1, dim, device=cuda).half()
    paged.append_kv8(x, x, ints([2 * bs], cuda, torch.int64), kc, vc, ks, vs)
    assert capi.device_error(0) == 4 and not kc.any() and not ks.any()
    paged.append_kv8(x, x, ints([0], cuda, torch.int64), kc, vc, ks, vs, freqs=angles(dim, 4, cuda), positions=ints([4], cuda, torch.int64))
    assert capi.device_error(0) == 4
    assert capi.device_error(0) == 0


# ---- attention --------------------------------------------------------------------

def make_cache(pool, kv_heads, bs, dim, kind, dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    top = TOP[kind]
    c = (torch.randn(pool, kv_heads, bs, dim, generator=gen, device=dev) * top / 4).clamp(-top, top)
    c = c.round().to(torch.int8) if kind == "int8" else c.to(CODE[kind])
    s = (4 / top) * torch.exp(0.5 * torch.randn(pool, kv_heads, generator=gen, device=dev))
    return c, s


def attend_ref(q, kc, vc, ks, vs, table, lens, starts, scale, out_eps, least=2.0 ** -24):
    """(o, bound) in 64 bits.  The bound: a weight rounded to 11 bits (2^-11) and the fp32 sums (2^-14) of sum p |v|, weights under
    2^-14 of the largest by 2^-24 each, the scores' fp32 sums (2^-18 of sum |q||k|), and the output's rounding (``least``: its smallest
    step)."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    hq, d = q.shape[1], q.shape[2]
    hk, bs = kc.shape[1], kc.shape[2]
    kb, vb = kc.view(torch.uint8), vc.view(torch.uint8)
    for r, n_all in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        n = b - a
        if n == 0 or n_all <= 0:
            continue
        rows = table[r, :-(-n_all // bs)].long()
        seen = torch.arange(n_all, device=q.device)[None, :] <= n_all - n + torch.arange(n, device=q.device)[:, None]
        for h in range(hk):
            k = (kb[rows, h].view(kc.dtype).double() * ks[rows, h].double()[:, None, None]).reshape(-1, d)[:n_all]
            v = (vb[rows, h].view(vc.dtype).double() * vs[rows, h].double()[:, None, None]).reshape(-1, d)[:n_all]
            g = slice(h * (hq // hk), (h + 1) * (hq // hk))
            x = q[a:b, g].double().transpose(0, 1)
            s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(seen.any(-1)[None, :, None], p, 0.0)
            o[a:b, g] = (p @ v).transpose(0, 1)
            size = p @ v.abs()
            score = (x.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
            lim = size * (2.0 ** -11 + 2.0 ** -14 + 2.0 ** -18 * score) + n_all * 2.0 ** -24 * v.abs().max()
            bound[a:b, g] = lim.transpose(0, 1)
    return o, bound + o.abs() * out_eps + least


def run_attend(cuda, kind, dtype, heads, kv_heads, dim, bs, lens, new, seed=0, view=False):
    rng = random.Random(seed)
    blocks = [-(-max(n, 0) // bs) for n in lens]
    pool = sum(blocks) + 2
    ids = list(range(pool))
    rng.shuffle(ids)
    width = max(blocks + [1]) + 1
    table = [[ids.pop() for _ in range(b)] + [-1] * (width - b) for b in blocks]
    kc, ks = make_cache(pool, kv_heads, bs, dim, kind, cuda, seed + 1)
    vc, vs = make_cache(pool, kv_heads, bs, dim, kind, cuda, seed + 2)
    # whatever lies past a request's end must not matter
    for r, n in enumerate(lens):
        if n > 0 and n % bs:
            for c in (kc, vc):
                c.view(torch.uint8)[table[r][n // bs], :, n % bs:] = 0x7F if kind == "e4m3" else 0x80
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    gen = torch.Generator(device=cuda).manual_seed(seed + 3)
    t = starts[-1]
    if view:
        q = torch.randn(t, heads + 2 * kv_heads, dim, generator=gen, device=cuda).to(HALF[dtype])[:, :heads]
    else:
        q = torch.randn(t, heads, dim, generator=gen, device=cuda).to(HALF[dtype])
    tb = ints(table, cuda)
    ws = paged.attend_workspace(len(lens), max(new), heads, kv_heads, dim, cuda)
    got = paged.attend_kv8(q, kc, vc, ks, vs, tb, ints(lens, cuda), ints(starts, cuda), max(new), max(lens), workspace=ws)
    again = paged.attend_kv8(q, kc, vc, ks, vs, tb, ints(lens, cuda), ints(starts, cuda), max(new), max(lens), workspace=ws)
    want, bound = attend_ref(q, kc, vc, ks, vs, tb, lens, starts, 1 / math.sqrt(dim), 2.0 ** -11 if dtype == "f16" else 2.0 ** -8)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst error / bound {(err / bound).max().item()}"
    assert torch.equal(got, again), "the same call twice"
    assert capi.device_error(0) == 0
    return got


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,bs", [("f16", 8, 8, 64, 16), ("bf16", 8, 2, 128, 32), ("f16", 64, 8, 128, 64),
                                                         ("bf16", 32, 2, 256, 128), ("f16", 3, 1, 256, 16), ("f16", 40, 1, 128, 128)])
def test_attend_single_tokens(cuda, kind, dtype, heads, kv_heads, dim, bs):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 500, 1023, 2049]
    run_attend(cuda, kind, dtype, heads, kv_heads, dim, bs, lens, [1] * len(lens), seed=dim + bs, view=bs == 64)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,bs", [("f16", 4, 4, 64, 64), ("bf16", 8, 2, 128, 16), ("f16", 16, 2, 128, 64),
                                                         ("bf16", 8, 2, 256, 32), ("f16", 7, 1, 128, 128)])
def test_attend_prompts(cuda, kind, dtype, heads, kv_heads, dim, bs):
    """New tokens from one to several hundred, alone and over a cached prefix, single tokens among them."""
    new = [1, 2, 5, 16, 33, 129, 300, 64]
    lens = [1, 2, 77, 16, 40, 129, 811, 64 + 3 * bs]
    run_attend(cuda, kind, dtype, heads, kv_heads, dim, bs, lens, new, seed=dim + 2 * bs, view=bs == 64)


def test_attend_empty_rows(cuda):
    """Requests without new tokens, an empty request with one padded query (zeros), and queries that outnumber the positions."""
    got = run_attend(cuda, "e4m3", "f16", 8, 2, 128, 16, [40, 0, 33, 3, 0], [1, 1, 0, 5, 0], seed=5)
    assert not got[1].any()
    assert not got[2:4].any() and bool(got[4:].abs().amax(-1).all())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attend_long(cuda, kind):
    """One and two requests long enough that the work of a head is split."""
    run_attend(cuda, kind, "bf16", 8, 1, 128, 64, [70001], [1], seed=3)
    run_attend(cuda, kind, "f16", 8, 2, 128, 16, [30000, 7], [3, 1], seed=4)


def test_attend_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 codes, the request's blocks at its far end."""
    bs, heads, dim = 128, 8, 128
    pool = (1 << 32) // (bs * heads * dim) + 40
    kc = torch.zeros(pool, heads, bs, dim, dtype=torch.int8, device=cuda)
    vc = torch.zeros(pool, heads, bs, dim, dtype=torch.int8, device=cuda)
    ks, vs = torch.full((pool, heads), 0.01, device=cuda), torch.full((pool, heads), 0.02, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(9)
    n = 300
    ids = [pool - 1, pool - 17, pool - 5]
    x = torch.randn(n, 3 * heads, dim, generator=gen, device=cuda).half()
    q, k, v = x[:, :heads], x[:, heads:2 * heads], x[:, 2 * heads:]
    slots = ints([ids[p // bs] * bs + p % bs for p in range(n)], cuda, torch.int64)
    paged.append_kv8(k, v, slots, kc, vc, ks, vs)
    table = ints([ids], cuda)
    for first in (0, n - 1):
        got = paged.attend_kv8(q[first:], kc, vc, ks, vs, table, ints([n], cuda), ints([0, n - first], cuda), n - first, n)
        want, bound = attend_ref(q[first:], kc, vc, ks, vs, table, [n], [0, n - first], 1 / math.sqrt(dim), 2.0 ** -11)
        assert bool(((got.double() - want).abs() <= bound).all())
    assert capi.device_error(0) == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attend_scales_far_apart(cuda, kind):
    """Values of blocks 2^30 apart, a block of zeros and a tiny one: the weights stay those of the softmax."""
    bs, dim = 16, 128
    kc, _ = make_cache(5, 1, bs, dim, kind, cuda, 1)
    vc, _ = make_cache(5, 1, bs, dim, kind, cuda, 2)
    ks = torch.full((5, 1), 1.0 / TOP[kind], device=cuda)
    vs = torch.tensor([[2.0 ** -30], [1.0], [0.0], [2.0 ** -12], [2.0 ** -90]], device=cuda) / TOP[kind]
    vc.view(torch.uint8)[2] = 0
    q = torch.randn(1, 4, dim, device=cuda).half()
    for table, n in (([[0, 1, 2, 3]], 64), ([[0, 2]], 32), ([[4, 4]], 30)):
        t = ints(table, cuda)
        got = paged.attend_kv8(q.bfloat16(), kc, vc, ks, vs, t, ints([n], cuda), ints([0, 1], cuda), 1, n)
        want, bound = attend_ref(q.bfloat16(), kc, vc, ks, vs, t, [n], [0, 1], 1 / math.sqrt(dim), 2.0 ** -8, least=2.0 ** -126)
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("new", [1, 40])
def test_attend_marked_block_reaches_only_who_sees_it(cuda, new):
    bs, dim = 16, 128
    kc, ks = make_cache(8, 2, bs, dim, "int8", cuda, 1)
    vc, vs = make_cache(8, 2, bs, dim, "int8", cuda, 2)
    table = ints([[0, 1, 2, 3], [4, 5, 6, 7]], cuda)
    ks[3, 0] = math.nan
    vs[6, 1] = math.nan
    q = torch.randn(2 * new, 4, dim, device=cuda).half()
    got = paged.attend_kv8(q, kc, vc, ks, vs, table, ints([64, 64], cuda), ints([0, new, 2 * new], cuda), new, 64)
    pos = torch.arange(64 - new, 64, device=cuda)
    bad = torch.isnan(got).all(-1)
    assert torch.equal(bad, torch.isnan(got).any(-1))
    assert torch.equal(bad[:new, :2], (pos >= 48)[:, None].expand(-1, 2)) and not bad[:new, 2:].any()
    assert torch.equal(bad[new:, 2:], (pos >= 32)[:, None].expand(-1, 2)) and not bad[new:, :2].any()


def test_attend_large_and_tiny_queries(cuda):
    """bf16 queries far outside fp16's range: the softmax scale brings the scores back."""
    kc, ks = make_cache(4, 2, 32, 64, "e4m3", cuda, 1)
    vc, vs = make_cache(4, 2, 32, 64, "e4m3", cuda, 2)
    table, lens = ints([[2, 0, 1, 3]], cuda), [101]
    for size in (2.0 ** 40, 2.0 ** -60):
        q = (torch.randn(1, 4, 64, device=cuda) * size).bfloat16()
        scale = 0.125 / size
        got = paged.attend_kv8(q, kc, vc, ks, vs, table, ints(lens, cuda), ints([0, 1], cuda), 1, 101, softmax_scale=scale)
        want, bound = attend_ref(q, kc, vc, ks, vs, table, lens, [0, 1], scale, 2.0 ** -8)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_attend_bad_block(cuda):
    """A table entry out of range is read as block 0 and reported."""
    kc, ks = make_cache(2, 1, 16, 64, "int8", cuda, 1)
    q = torch.randn(1, 1, 64, device=cuda).half()
    got = paged.attend_kv8(q, kc, kc, ks, ks, ints([[2]], cuda), ints([5], cuda), ints([0, 1], cuda), 1, 5)
    want = paged.attend_kv8(q, kc, kc, ks, ks, ints([[0]], cuda), ints([5], cuda), ints([0, 1], cuda), 1, 5)
    assert torch.equal(got, want)
    assert capi.device_error(0) == 4
    assert capi.device_error(0) == 0


def test_side_stream_and_graph(cuda):
    """The three calls on a side stream and replayed from a graph give the same bits."""
    bs, hk, dim, requests = 16, 2, 64, 3
    context, new = ints([5, 16, 40], cuda), ints([1, 1, 1], cuda)
    free = torch.arange(20, dtype=torch.int32, device=cuda)
    kc, ks = make_cache(20, hk, bs, dim, "e4m3", cuda, 1)
    vc, vs = make_cache(20, hk, bs, dim, "e4m3", cuda, 2)
    table = ints([[10, -1, -1, -1], [11, -1, -1, -1], [12, 13, 14, -1]], cuda)
    x = torch.randn(requests, 8, dim, device=cuda).half()
    f = angles(dim, 64, cuda)
    ws = paged.attend_workspace(requests, 1, 4, hk, dim, cuda)
    head = ints([0], cuda)

    def step():
        t = paged.build_tables(context, new, table, free, head, bs, requests)
        q = paged.append_kv8(x[:, 4:6], x[:, 6:], t.slots, kc, vc, ks, vs, q=x[:, :4], freqs=f, positions=t.positions)
        return paged.attend_kv8(q, kc, vc, ks, vs, table, t.seq_lens, t.query_starts, 1, 64, workspace=ws)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
