"""A batch of requests over a paged KV cache held in 8 bits.

GdsLLM serves one request at a time over a preallocated fp16 cache
(gdsllm/runtime/kv_cache.py:35-67).  Here requests of any lengths share one
pool of cache blocks.  A step is

    build_tables   block table, sequence lengths, positions and cache slots of
                   the step's new tokens, on the GPU from the request lengths
    append_kv8     per layer: RoPE of q and k, K and V into the cache as 8-bit
                   codes with one fp32 scale per (block, KV head)
    attend_kv8     per layer: attention of the new tokens over the cache

and ``sampling.sample`` picks the tokens.  The cache of one layer is ``k_cache``
and ``v_cache`` [blocks, kv_heads, block_size, head_dim], int8 or
float8_e4m3fn, with ``k_scale`` and ``v_scale`` [blocks, kv_heads] fp32; a value
is code * scale.  block_size is 16, 32, 64 or 128, head_dim 64, 128 or 256.
Activations are fp16 or bf16.

Every function launches on the current stream of its tensors' device, raises
``ValueError`` for arguments it does not take and ``GdsqError`` for a non-OK
status, and is safe to capture in a CUDA graph (lengths live on the device).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._native import ext


class StepTables(NamedTuple):
    """What ``build_tables`` makes for one step of R requests and T tokens."""
    seq_lens: torch.Tensor      # int32 [R]: tokens of each request after the step
    query_starts: torch.Tensor  # int32 [R + 1]: where each request's new tokens begin
    positions: torch.Tensor     # int64 [T]
    slots: torch.Tensor         # int64 [T]: block * block_size + offset; -1 = none
    free_head: torch.Tensor     # int32 [1]: the queue's head after the step


def build_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                 free_blocks: torch.Tensor, free_head: torch.Tensor, block_size: int, num_tokens: int,
                 out: StepTables | None = None) -> StepTables:
    """The step's tables: request r holds ``context_lens[r]`` tokens and gets
    ``new_lens[r]`` more (int32 [R], on the GPU).  ``block_table`` [R, W] int32
    gets its new entries in place, from ``free_blocks[free_head:]`` in request
    order.  ``num_tokens`` sizes the per-token outputs; tokens past the sum of
    ``new_lens`` get slot -1.  A row or a queue that is too short sets device
    error bit 4 (``capi.device_error``).  ``out`` takes the results in place of
    new tensors; none of them may share memory with an input, so a loop that
    feeds ``seq_lens`` and ``free_head`` back takes turns between two."""
    t = ext().build_tables(context_lens, new_lens, block_table, free_blocks, free_head, block_size, num_tokens, out)
    return StepTables(*t) if out is None else out


def append_kv8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               k_scale: torch.Tensor, v_scale: torch.Tensor, *, q: torch.Tensor | None = None,
               freqs: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes k and v [T, kv_heads, dim] (any token and head strides that are
    multiples of 8) into the cache slots ``slots`` [T] int64, in place.  The new
    tokens of one block must be adjacent, as ``build_tables`` orders them.
    With ``freqs`` (fp32 [positions, dim / 2, 2], ``view_as_real`` of GdsLLM's
    ``freqs_cis``) k is rotated by ``positions`` [T] first, and so is q
    [T, heads, dim], which is returned ([T, heads, dim], contiguous)."""
    return ext().append_kv8(k, v, slots, k_cache, v_cache, k_scale, v_scale, q, freqs, positions, q_out)


def attend_workspace(num_requests: int, max_query_len: int, num_heads: int, num_kv_heads: int, head_dim: int,
                     device) -> torch.Tensor:
    """A zeroed workspace for ``attend_kv8`` calls up to these sizes.  Keep it
    from call to call; calls that may run at the same time need one each."""
    return ext().attend_workspace(num_requests, max_query_len, num_heads, num_kv_heads, head_dim, device)


def attend_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, query_starts: torch.Tensor,
               max_query_len: int, max_seq_len: int | None = None, *, softmax_scale: float | None = None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens q [T, heads, dim] over the cache: request
    r's tokens are ``query_starts[r]:query_starts[r + 1]``, the last of its
    ``seq_lens[r]``, and each sees the positions up to its own.  Heads share KV
    heads in order (heads a multiple of kv_heads).  ``max_query_len`` is the
    largest number of new tokens of a request, which the host does not see: it
    chooses the kernel, and a request with more is only slower.  Nothing
    depends on ``max_seq_len``, which callers that have it may give.  Returns
    [T, heads, dim]; a query that sees nothing gives zeros, as does a token behind
    the last request's.  ``workspace``: see ``attend_workspace``
    (allocated for the call when not given)."""
    return ext().attend_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_starts, max_query_len,
                            max_seq_len, softmax_scale, out, workspace)
