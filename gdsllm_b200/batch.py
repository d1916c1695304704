"""A LLaMA model serving a batch of requests over the paged 8-bit cache.

GdsLLM runs one request at a time (the ``batch == 1`` asserts of
gdsllm/runtime/scheduler.py:137,318) over an fp16 cache and samples on the
host (gdsllm/engine.py:47-95).  ``BatchLlama`` takes the same layer dicts as
``decode_step.GraphDecodeStep`` and serves requests of any lengths together;
one ``step`` runs

    build_tables                       block table, positions, slots
    embedding
    per layer:  add_rmsnorm, q/k/v, append_kv8 (RoPE and the 8-bit cache
                write), attend_kv8, o, add_rmsnorm, gate/up, silu_mul, down
    add_rmsnorm, lm_head of each request's last token

and ``sample`` picks the tokens.  Up to 16 tokens a step the projections are
the fused dequant-GEMVs; longer steps (prompts) dequantize a matrix and
multiply, as GdsLLM's prefill does (gdsllm/runtime/llama.py:144-166).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import capi, paged, sampling
from .decode_step import _gguf_matrix, _Layer, _gemv

GEMV_MAX_TOKENS = 16  # GDSQ_MAX_BATCH


class BatchLlama:
    """``layers`` are the per-layer tensor dicts of ``transformer_block``
    (Q4_0 / Q8_0 projections, fp16 norms), ``embed`` the embed_tokens dict,
    ``final_norm`` the fp16 norm weight, ``lm_head`` the GGUF head entry and
    ``freqs_cis`` the complex RoPE table.  ``max_requests`` rows share
    ``num_blocks`` cache blocks of ``block_size`` tokens per layer, held as
    ``cache_dtype`` (float8_e4m3fn or int8)."""

    def __init__(self, layers, embed: dict, final_norm: torch.Tensor, lm_head: dict, freqs_cis: torch.Tensor,
                 num_heads: int, num_kv_heads: int, rms_norm_eps: float, max_requests: int, num_blocks: int,
                 block_size: int = 64, cache_dtype: torch.dtype = torch.float8_e4m3fn):
        self.layers = [_Layer(t, i) for i, t in enumerate(layers)]
        if not self.layers:
            raise ValueError("BatchLlama: no layers")
        first = self.layers[0]
        self.hidden, self.num_heads, self.num_kv_heads = first.q[3], int(num_heads), int(num_kv_heads)
        self.head_dim = self.hidden // self.num_heads
        self.eps = float(rms_norm_eps)
        if first.q[2] != self.num_heads * self.head_dim or first.k[2] != self.num_kv_heads * self.head_dim:
            raise ValueError(f"BatchLlama: q has {first.q[2]} rows, k {first.k[2]}; {num_heads} and {num_kv_heads} heads "
                             f"of {self.head_dim} expected")
        dev = self.device = first.in_norm.device
        self.freqs = torch.view_as_real(freqs_cis).contiguous()
        w = embed["model.embed_tokens.weight"]
        self.embed = ("f16", w, *map(int, w.shape)) if isinstance(w, torch.Tensor) else _gguf_matrix(w, "model.embed_tokens.weight")
        self.final_norm = final_norm
        self.lm = _gguf_matrix(lm_head, "lm_head")
        shape = (len(self.layers), num_blocks, self.num_kv_heads, block_size, self.head_dim)
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=torch.uint8, device=dev).view(cache_dtype) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
        self.block_size, self.max_requests = int(block_size), int(max_requests)
        self.max_seq = int(self.freqs.shape[0])
        self.table = torch.full((max_requests, -(-self.max_seq // block_size)), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(num_blocks, dtype=torch.int32, device=dev)
        self.free_head = torch.zeros(1, dtype=torch.int32, device=dev)
        self.lengths = [0] * self.max_requests  # the host's copy: it sizes the launches
        self.blocks_left = int(num_blocks)
        self.workspace = paged.attend_workspace(max_requests, self.max_seq, self.num_heads, self.num_kv_heads, self.head_dim, dev)

    def _embed(self, ids: torch.Tensor) -> torch.Tensor:
        kind, table, rows, cols = self.embed
        return table[ids] if kind == "f16" else capi.dequant_rows(kind, table, rows, cols, ids)

    def _project(self, mats, x: torch.Tensor) -> list[torch.Tensor]:
        """Each matrix's output [tokens, rows]."""
        out = []
        for fmt, w, n, k in mats:
            if x.shape[0] <= GEMV_MAX_TOKENS:
                y = torch.empty(x.shape[0], n, dtype=torch.float16, device=self.device)
                _gemv(fmt, w, x, n, k, y)
            else:
                y = F.linear(x, (capi.dequant_q4_0 if fmt == "q4_0" else capi.dequant_q8_0)(w).view(n, k))
            out.append(y)
        return out

    def step(self, new_tokens: list[list[int]]) -> torch.Tensor:
        """Appends ``new_tokens[r]`` (may be empty) to request r and returns
        the logits [max_requests, vocab] after its last token (a request
        without new tokens: those of the step's last token, to be ignored).
        A step that raises leaves every request as it was: the host's lengths
        and the queue of free blocks move when all its work is launched, and
        tokens written past a request's length are written again."""
        if len(new_tokens) != self.max_requests:
            raise ValueError(f"BatchLlama: {len(new_tokens)} lists for {self.max_requests} requests")
        counts = [len(t) for t in new_tokens]
        tokens = sum(counts)
        if tokens == 0:
            raise ValueError("BatchLlama: no new token in the step")
        if not all(0 <= i < self.embed[2] for t in new_tokens for i in t):
            raise ValueError(f"BatchLlama: token outside the vocabulary of {self.embed[2]}")
        after = [a + b for a, b in zip(self.lengths, counts)]
        if max(after) > self.max_seq:
            raise ValueError(f"BatchLlama: {max(after)} positions, {self.max_seq} in the RoPE table")
        bs = self.block_size
        taken = sum(-(-b // bs) - -(-a // bs) for a, b in zip(self.lengths, after))
        if taken > self.blocks_left:
            raise ValueError(f"BatchLlama: {taken} cache blocks needed, {self.blocks_left} free")
        ids, context, new = (torch.tensor(v, dtype=t, device=self.device) for v, t in (
            ([i for t in new_tokens for i in t], torch.int64), (self.lengths, torch.int32), (counts, torch.int32)))
        t = paged.build_tables(context, new, self.table, self.free, self.free_head, bs, tokens)
        d = self.head_dim
        h = self._embed(ids)
        delta = None
        for i, lay in enumerate(self.layers):
            x = capi.add_rmsnorm(h, lay.in_norm, self.eps, delta=delta)
            q, k, v = (y.view(tokens, -1, d) for y in self._project([lay.q, lay.k, lay.v], x))
            cache = (self.k_cache[i], self.v_cache[i], self.k_scale[i], self.v_scale[i])
            q = paged.append_kv8(k, v, t.slots, *cache, q=q, freqs=self.freqs, positions=t.positions)
            a = paged.attend_kv8(q, *cache, self.table, t.seq_lens, t.query_starts, max(counts), max(after), workspace=self.workspace)
            delta, = self._project([lay.o], a.view(tokens, -1))
            x = capi.add_rmsnorm(h, lay.post_norm, self.eps, delta=delta)
            delta, = self._project([lay.down], capi.silu_mul(*self._project([lay.gate, lay.up], x)))
        last = (t.query_starts[1:].long() - 1).clamp_min(0)
        x = capi.add_rmsnorm(h[last].contiguous(), self.final_norm, self.eps, delta=delta[last].contiguous())
        logits, = self._project([self.lm], x)
        self.free_head = t.free_head
        self.blocks_left -= taken
        self.lengths = after
        return logits

    def release(self, request: int) -> None:
        """Frees a finished request's cache blocks for the requests to come."""
        n = -(-self.lengths[request] // self.block_size)
        if n:
            # the blocks taken so far are behind the queue's head: put these back in front of it
            head = self.free_head.long()
            at = head - n + torch.arange(n, device=self.device)
            self.free[at] = self.table[request, :n]
            self.free_head = (head - n).to(torch.int32)
            self.blocks_left += n
        self.lengths[request] = 0

    def generate(self, prompts: list[list[int]], new_tokens: int, *, temperature: float = 1.0, top_k: int = 0,
                 top_p: float = 1.0, min_p: float = 0.0, seed: int = 0):
        """The prompts (at most ``max_requests``) and ``new_tokens`` sampled
        tokens for each: (tokens int64, log-probabilities fp32), both
        [prompts, new_tokens] on the host.  The requests' blocks are free
        again afterwards."""
        if not 0 < len(prompts) <= self.max_requests or any(self.lengths) or not all(prompts):
            raise ValueError(f"BatchLlama: 1 to {self.max_requests} non-empty prompts, with no request being served")
        if new_tokens < 0:
            raise ValueError(f"BatchLlama: {new_tokens} new tokens")
        if new_tokens == 0:
            return torch.empty(len(prompts), 0, dtype=torch.int64), torch.empty(len(prompts), 0)
        n, dev = len(prompts), self.device
        gen = torch.Generator(device=dev).manual_seed(seed)
        rows = dict(temperature=torch.full((n,), temperature, device=dev), top_k=torch.full((n,), top_k, dtype=torch.int32, device=dev),
                    top_p=torch.full((n,), top_p, device=dev), min_p=torch.full((n,), min_p, device=dev))
        idle = [[]] * (self.max_requests - n)
        step, tokens, logprobs = [list(p) for p in prompts], [], []
        try:
            for _ in range(new_tokens):
                logits = self.step(step + idle)
                t, lp = sampling.sample(logits[:n], torch.rand(n, generator=gen, device=dev), **rows)
                tokens.append(t.cpu())
                logprobs.append(lp.cpu())
                step = [[i] for i in tokens[-1].tolist()]
        finally:
            for r in range(n):
                self.release(r)
        return torch.stack(tokens, 1), torch.stack(logprobs, 1)
