"""What the batched-serving entry points refuse, without a GPU: the C ABI
checks every argument before any CUDA call, the Python functions raise
ValueError for tensors they do not take."""
from __future__ import annotations

import pytest
import torch

from gdsllm_b200 import paged, sampling
from gdsllm_b200._native import lib

P = 0x10000  # never dereferenced


def tables(l, requests=1, width=1, block=16, tokens=1, head=P, head_out=2 * P, table=P, slots=P):
    return l.gdsq_build_tables(P, P, requests, table, width, P, 1, head, block, tokens, P, P, P, slots, head_out, None)


def append(l, elem=0, k=P, stride=64, freqs=None, q=None, q_out=None, positions=None, tokens=1, kv_heads=1, dim=64, kind=0, cache=P, block=16):
    return l.gdsq_append_kv8(elem, q, stride, 64, k, stride, 64, P, stride, 64, q_out, freqs, 8, positions, P, tokens, 1, kv_heads, dim,
                             kind, cache, P, P, P, 4, block, None)


def attend(l, q=P, elem=0, stride=64, cache=P, kind=0, block=16, requests=1, tokens=1, longest=1, heads=2, kv_heads=1, dim=64, out=P):
    return l.gdsq_attend_kv8(q, elem, stride, 64, cache, P, kind, P, P, 4, block, P, 4, P, P, requests, tokens, longest, 64, heads,
                             kv_heads, dim, 0.1, out, None, 0, None)


def sample(l, elem=0, logits=P, rows=1, vocab=10, tokens=P, u=P):
    return l.gdsq_sample(elem, logits, vocab, rows, vocab, u, None, None, None, None, tokens, None, None)


@pytest.mark.parametrize("call,status,text", [
    (lambda l: tables(l, requests=0), 1, b"requests 0"),
    (lambda l: tables(l, requests=16385), 1, b"16384"),
    (lambda l: tables(l, block=0), 1, b"block"),
    (lambda l: tables(l, tokens=-1), 1, b"tokens -1"),
    (lambda l: tables(l, table=None), 1, b"null"),
    (lambda l: tables(l, head_out=P), 1, b"free_head_out"),
    (lambda l: tables(l, slots=P + 4), 2, b"8-byte"),
    (lambda l: append(l, elem=1), 1, b"elem_type"),
    (lambda l: append(l, kind=2), 1, b"cache_type"),
    (lambda l: append(l, dim=96), 3, b"head_dim 96"),
    (lambda l: append(l, block=48), 3, b"block_size 48"),
    (lambda l: append(l, kv_heads=0), 1, b"kv heads 0"),
    (lambda l: append(l, k=None), 1, b"null"),
    (lambda l: append(l, freqs=P), 1, b"null"),
    (lambda l: append(l, q=P, q_out=P), 1, b"q and q_out"),
    (lambda l: append(l, freqs=P, positions=P, q=P), 1, b"q and q_out"),
    (lambda l: append(l, stride=68), 2, b"multiples of 8"),
    (lambda l: append(l, cache=P + 64), 2, b"128-byte"),
    (lambda l: attend(l, elem=1), 1, b"elem_type"),
    (lambda l: attend(l, kind=-1), 1, b"cache_type"),
    (lambda l: attend(l, heads=3, kv_heads=2), 1, b"multiple of kv heads"),
    (lambda l: attend(l, dim=80), 3, b"head_dim 80"),
    (lambda l: attend(l, block=256), 3, b"block_size 256"),
    (lambda l: attend(l, requests=65536), 1, b"requests 65536"),
    (lambda l: attend(l, longest=-1), 1, b"negative"),
    (lambda l: attend(l, q=None), 1, b"null"),
    (lambda l: attend(l, q=P + 2), 2, b"16-byte"),
    (lambda l: attend(l, cache=P + 16), 2, b"128-byte"),
    (lambda l: sample(l, elem=2), 1, b"elem_type"),
    (lambda l: sample(l, vocab=0), 1, b"vocab 0"),
    (lambda l: sample(l, vocab=524289), 1, b"vocab 524289"),
    (lambda l: sample(l, u=None), 1, b"null"),
    (lambda l: sample(l, logits=P + 1), 2, b"alignment"),
    (lambda l: sample(l, tokens=P + 4), 2, b"8-byte"),
])
def test_c_entry_refuses(call, status, text):
    l = lib()
    assert call(l) == status
    assert text in l.gdsq_last_error(), l.gdsq_last_error()


@pytest.mark.parametrize("call", [lambda l: append(l, tokens=0), lambda l: attend(l, tokens=0), lambda l: attend(l, requests=0),
                                  lambda l: attend(l, longest=0), lambda l: sample(l, rows=0)])
def test_nothing_to_do_is_ok(call):
    assert call(lib()) == 0


def cache(dtype=torch.int8, heads=2, bs=16, dim=64):
    c = torch.zeros(4, heads, bs, dim, dtype=dtype)
    return c, c.clone(), torch.zeros(4, heads), torch.zeros(4, heads)


def test_python_refuses():
    kc, vc, ks, vs = cache()
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    bad = [
        ("k: fp16 or bf16", lambda: paged.append_kv8(x.float(), x, slots, kc, vc, ks, vs)),
        ("v: fp16 or bf16", lambda: paged.append_kv8(x, x.bfloat16(), slots, kc, vc, ks, vs)),
        ("k: expected", lambda: paged.append_kv8(x[:, :1], x, slots, kc, vc, ks, vs)),
        ("k has 3 tokens, v 2", lambda: paged.append_kv8(x, x[:2], slots, kc, vc, ks, vs)),
        ("slots: expected", lambda: paged.append_kv8(x, x, slots.int(), kc, vc, ks, vs)),
        ("the cache is int8 or", lambda: paged.append_kv8(x, x, slots, kc.half(), vc, ks, vs)),
        ("k_cache and v_cache", lambda: paged.append_kv8(x, x, slots, kc, vc[:2], ks, vs)),
        ("the scales are", lambda: paged.append_kv8(x, x, slots, kc, vc, ks.half(), vs)),
        ("q is only rotated", lambda: paged.append_kv8(x, x, slots, kc, vc, ks, vs, q=x)),
        ("freqs needs positions", lambda: paged.append_kv8(x, x, slots, kc, vc, ks, vs, freqs=torch.zeros(8, 32, 2))),
        ("freqs: contiguous", lambda: paged.append_kv8(x, x, slots, kc, vc, ks, vs, freqs=torch.zeros(8, 64, 2), positions=slots)),
        ("k: expected", lambda: paged.append_kv8(x.transpose(1, 2), x, slots, kc, vc, ks, vs)),
        ("q: fp16 or bf16", lambda: paged.attend_kv8(x.float(), kc, vc, ks, vs, i32(1, 4), i32(1), i32(2), 3)),
        ("block_table", lambda: paged.attend_kv8(x, kc, vc, ks, vs, i32(2, 4), i32(1), i32(2), 3)),
        ("out: contiguous", lambda: paged.attend_kv8(x, kc, vc, ks, vs, i32(1, 4), i32(1), i32(2), 3, out=x.bfloat16())),
        ("block_table", lambda: paged.build_tables(i32(2), i32(2), i32(3, 4), i32(9), i32(1), 16, 4)),
        ("logits:", lambda: sampling.sample(torch.zeros(5), torch.zeros(1))),
        ("logits:", lambda: sampling.sample(torch.zeros(2, 5, dtype=torch.float64), torch.zeros(2))),
        ("logits:", lambda: sampling.sample(torch.zeros(5, 2).t(), torch.zeros(2))),
    ]
    for text, call in bad:
        with pytest.raises(ValueError, match=text):
            call()
