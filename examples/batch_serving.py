#!/usr/bin/env python3
"""Serves a batch of prompts of different lengths on a small LLaMA with random
Q4_0 weights: step tables, the 8-bit paged cache, attention over it and
sampling, as ``gdsllm_b200.batch.BatchLlama`` runs them.

    python examples/batch_serving.py [--requests 6] [--tokens 32] [--cache e4m3|int8]
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import gdsllm_b200  # noqa: E402
from gdsllm_b200 import capi, synth  # noqa: E402
from gdsllm_b200.batch import BatchLlama  # noqa: E402


def random_model(layers: int, hidden: int, heads: int, kv_heads: int, ffn: int, vocab: int, device, seed: int = 0, max_seq: int = 4096):
    """(layers, embed, final norm, lm_head, freqs_cis) of a LLaMA with random weights, in GdsLLM's forms."""
    ext = gdsllm_b200.ext()
    head_dim = hidden // heads
    gen = torch.Generator(device=device).manual_seed(seed)

    def gguf(kind, n, k, s):
        raw = (synth.q4_0_weight if kind == "q4_0" else synth.q8_0_weight)(n, k, seed=seed * 1000 + s, device=device)
        return {"buffer": ext.handle_from_tensor(raw.reshape(-1)), "shape": [n, k], "gguf_type": kind, "offset": 0}

    def norm():
        return (1 + 0.1 * torch.randn(hidden, generator=gen, device=device)).half()

    dims = {"self_attn.q_proj": (hidden, hidden), "self_attn.k_proj": (kv_heads * head_dim, hidden),
            "self_attn.v_proj": (kv_heads * head_dim, hidden), "self_attn.o_proj": (hidden, hidden), "mlp.gate_proj": (ffn, hidden),
            "mlp.up_proj": (ffn, hidden), "mlp.down_proj": (hidden, ffn)}
    out = []
    for i in range(layers):
        t = {f"{name}.weight": gguf("q4_0", n, k, 10 * i + j) for j, (name, (n, k)) in enumerate(dims.items())}
        t["input_layernorm.weight"], t["post_attention_layernorm.weight"] = norm(), norm()
        out.append(t)
    embed = {"model.embed_tokens.weight": (0.02 * torch.randn(vocab, hidden, generator=gen, device=device)).half()}
    angle = torch.outer(torch.arange(max_seq, device=device).float(),
                        10000.0 ** (-torch.arange(0, head_dim, 2, device=device).float() / head_dim))
    return out, embed, norm(), gguf("q8_0", vocab, hidden, 9999), torch.polar(torch.ones_like(angle), angle)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--cache", choices=("e4m3", "int8"), default="e4m3")
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    heads, kv_heads, vocab = 16, 4, 32000
    layers, embed, norm, head, freqs = random_model(4, 2048, heads, kv_heads, 5504, vocab, dev)
    model = BatchLlama(layers, embed, norm, head, freqs, heads, kv_heads, 1e-5, max_requests=a.requests, num_blocks=64 * a.requests,
                       cache_dtype=torch.int8 if a.cache == "int8" else torch.float8_e4m3fn)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, vocab, (int(n),), generator=gen).tolist() for n in torch.randint(1, 400, (a.requests,), generator=gen)]
    for _ in range(2):  # the second run is warm
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        tokens, logprobs = model.generate(prompts, a.tokens, temperature=0.8, top_k=50, top_p=0.95, seed=3)
        torch.cuda.synchronize()
        seconds = time.perf_counter() - t0
    for p, t, lp in zip(prompts, tokens, logprobs):
        print(f"prompt of {len(p):3d} tokens -> {t[:8].tolist()} ...  mean log-probability {lp.mean():.3f}")
    print(f"{a.requests} requests, {a.tokens} tokens each: {a.requests * a.tokens / seconds:.0f} tokens/s, device error {capi.device_error(0)}")


if __name__ == "__main__":
    main()
