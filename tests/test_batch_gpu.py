"""The batch path (gdsllm_b200.batch) against a plain LLaMA forward in 32 bits
over exactly dequantized weights and an unrounded cache."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from gdsllm_b200 import capi
from gdsllm_b200.batch import BatchLlama
from gdsllm_b200.decode_step import _gguf_matrix

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("batch_serving", Path(__file__).resolve().parents[1] / "examples" / "batch_serving.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)

SHAPE = dict(layers=2, hidden=512, heads=4, kv_heads=2, ffn=1536, vocab=2048)


def dense(entry):
    fmt, raw, n, k = _gguf_matrix(entry, "weight")
    return (capi.dequant_q4_0 if fmt == "q4_0" else capi.dequant_q8_0)(raw).view(n, k).float()


def plain_logits(layers, embed, norm, head, freqs, tokens, eps=1e-5):
    """Logits after the last of ``tokens``: one causal forward in fp32."""
    def rms(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.float()

    heads, kv = SHAPE["heads"], SHAPE["kv_heads"]
    x = embed["model.embed_tokens.weight"][tokens].float()
    n = len(tokens)
    d = x.shape[1] // heads

    def turn(v):
        z = torch.view_as_complex(v.reshape(n, -1, d // 2, 2).contiguous()) * freqs[:n, None]
        return torch.view_as_real(z).flatten(2)
    hidden = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
    for t in layers:
        y = rms(x, t["input_layernorm.weight"])
        q, k, v = (y @ dense(t[f"self_attn.{p}_proj.weight"]).T for p in "qkv")
        q, k, v = turn(q), turn(k), v.view(n, kv, d)
        k, v = k.repeat_interleave(heads // kv, 1), v.repeat_interleave(heads // kv, 1)
        s = torch.einsum("ihd,jhd->hij", q, k) / d ** 0.5
        a = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(hidden, -torch.inf), -1), v)
        x = x + a.reshape(n, -1) @ dense(t["self_attn.o_proj.weight"]).T
        y = rms(x, t["post_attention_layernorm.weight"])
        g = torch.nn.functional.silu(y @ dense(t["mlp.gate_proj.weight"]).T) * (y @ dense(t["mlp.up_proj.weight"]).T)
        x = x + g @ dense(t["mlp.down_proj.weight"]).T
    return rms(x[-1], norm) @ dense(head).T


@pytest.fixture(scope="module")
def model(cuda):
    return example.random_model(device=cuda, seed=1, max_seq=512, **SHAPE)


# fp16 activations give about 2^-10 per operation; a cache code is off by 1/254 of its block's largest value at most (int8: about 1 %
# of a typical value) or by 2^-4 of itself (e4m3: 2 % in the mean).  Averaged over keys and layers, the logits' relative error (2-norm)
# has to stay under 3 % and 10 %.
@pytest.mark.parametrize("cache,bound", [(torch.int8, 0.03), (torch.float8_e4m3fn, 0.10)])
def test_batch_matches_plain_forward(cuda, model, cache, bound):
    b = BatchLlama(*model, SHAPE["heads"], SHAPE["kv_heads"], 1e-5, max_requests=4, num_blocks=64, block_size=16, cache_dtype=cache)
    gen = torch.Generator().manual_seed(2)
    text = [torch.randint(0, SHAPE["vocab"], (n,), generator=gen).tolist() for n in (3, 40, 0, 129)]
    seen = [list(t) for t in text]
    for step in range(4):
        new = text if step == 0 else [[int(torch.randint(0, SHAPE["vocab"], (1,), generator=gen))] if r != 1 or step > 1 else [] for r in range(4)]
        if step:
            for s, t in zip(seen, new):
                s += t
        logits = b.step(new).float()
        for r in range(4):
            if new[r]:
                want = plain_logits(*model, seen[r])
                err = ((logits[r] - want).norm() / want.norm()).item()
                assert err <= bound, (step, r, err)
    assert capi.device_error(0) == 0


def test_generate_and_release(cuda, model):
    """Greedy generation of a batch repeats itself, block by block, after its blocks went back."""
    b = BatchLlama(*model, SHAPE["heads"], SHAPE["kv_heads"], 1e-5, max_requests=3, num_blocks=12, block_size=16, cache_dtype=torch.int8)
    prompts = [[5, 6, 7], list(range(40)), [9] * 17]
    first, lp = b.generate(prompts, 10, temperature=0.0)
    assert first.shape == (3, 10) and bool((lp == 0).all())
    assert b.blocks_left == 12 and sorted(b.free.tolist()) == list(range(12))
    again, _ = b.generate(prompts, 10, temperature=0.0)
    assert torch.equal(first, again)
    sampled, lp = b.generate(prompts, 10, temperature=1.0, top_k=20, top_p=0.9, seed=4)
    assert bool((lp <= 0).all()) and bool((sampled >= 0).all())
    assert capi.device_error(0) == 0


def test_refusals(cuda, model):
    b = BatchLlama(*model, SHAPE["heads"], SHAPE["kv_heads"], 1e-5, max_requests=2, num_blocks=2, block_size=16)
    for bad in ([[1]], [[], []], [[1] * 40, []], [[1] * 600, []], [[-1], []], [[1], [2048]]):
        with pytest.raises(ValueError):
            b.step(bad)
    with pytest.raises(ValueError):
        b.generate([[1], [2], [3]], 1)
    with pytest.raises(ValueError):
        b.generate([[]], 1)
