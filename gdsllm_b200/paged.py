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

import math
from typing import NamedTuple

import torch

from ._native import check, lib

_ELEM = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 3}  # GDSQ_ELEM_*
_CACHE = {torch.int8: 0, torch.float8_e4m3fn: 1}                 # GDSQ_CACHE_*


class StepTables(NamedTuple):
    """What ``build_tables`` makes for one step of R requests and T tokens."""
    seq_lens: torch.Tensor      # int32 [R]: tokens of each request after the step
    query_starts: torch.Tensor  # int32 [R + 1]: where each request's new tokens begin
    positions: torch.Tensor     # int64 [T]
    slots: torch.Tensor         # int64 [T]: block * block_size + offset; -1 = none
    free_head: torch.Tensor     # int32 [1]: the queue's head after the step


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _ints(t: torch.Tensor, name: str, n: int, device, dtype=torch.int32) -> int:
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: expected {n} contiguous {dtype} on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def build_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                 free_blocks: torch.Tensor, free_head: torch.Tensor, block_size: int, num_tokens: int,
                 out: StepTables | None = None) -> StepTables:
    """The step's tables: request r holds ``context_lens[r]`` tokens and gets
    ``new_lens[r]`` more (int32 [R], on the GPU).  ``block_table`` [R, W] int32
    gets its new entries in place, from ``free_blocks[free_head:]`` in request
    order.  ``num_tokens`` sizes the per-token outputs; tokens past the sum of
    ``new_lens`` get slot -1.  A row or a queue that is too short sets device
    error bit 4 (``capi.device_error``)."""
    dev = context_lens.device
    r = context_lens.numel()
    _need(block_table.dim() == 2 and block_table.shape[0] == r, f"block_table {tuple(block_table.shape)} has not {r} rows")
    width = block_table.shape[1]
    if out is None:
        i32 = torch.empty(2 * r + 2, dtype=torch.int32, device=dev)
        i64 = torch.empty(2, num_tokens, dtype=torch.int64, device=dev)
        out = StepTables(i32[:r], i32[r:2 * r + 1], i64[0], i64[1], i32[2 * r + 1:])
    status = lib().gdsq_build_tables(
        _ints(context_lens, "context_lens", r, dev), _ints(new_lens, "new_lens", r, dev), r,
        _ints(block_table, "block_table", r * width, dev), width,
        _ints(free_blocks, "free_blocks", free_blocks.numel(), dev), free_blocks.numel(),
        _ints(free_head, "free_head", 1, dev), block_size, num_tokens,
        _ints(out.seq_lens, "out.seq_lens", r, dev), _ints(out.query_starts, "out.query_starts", r + 1, dev),
        _ints(out.positions, "out.positions", num_tokens, dev, torch.int64),
        _ints(out.slots, "out.slots", num_tokens, dev, torch.int64),
        _ints(out.free_head, "out.free_head", 1, dev), torch.cuda.current_stream(dev).cuda_stream)
    if status:
        check(status, "gdsq_build_tables")
    return out


def _cache(k_cache, v_cache, k_scale, v_scale):
    """Checks a layer's cache and returns its (type, blocks, heads, block size, dim)."""
    _need(k_cache.dtype in _CACHE, f"the cache is int8 or float8_e4m3fn, not {k_cache.dtype}")
    _need(k_cache.dim() == 4, f"the cache has 4 dimensions, not {k_cache.dim()}")
    shape = k_cache.shape
    if (v_cache.shape != shape or v_cache.dtype != k_cache.dtype or not k_cache.is_contiguous() or
            not v_cache.is_contiguous() or v_cache.device != k_cache.device):
        raise ValueError("k_cache and v_cache must be contiguous and alike")
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or s.shape != shape[:2] or not s.is_contiguous() or s.device != k_cache.device:
            raise ValueError(f"the scales are contiguous fp32 {tuple(shape[:2])}, got {tuple(s.shape)} {s.dtype}")
    return (_CACHE[k_cache.dtype], *shape)


def _rows(x: torch.Tensor, name: str, heads: int | None, dim: int, like: torch.Tensor, dtype=None):
    """[tokens, heads, dim] activations with a contiguous last dimension."""
    if x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads) or x.stride(2) != 1:
        raise ValueError(f"{name}: expected [tokens, {heads or 'heads'}, {dim}] with unit stride, got {tuple(x.shape)} "
                         f"strides {x.stride()}")
    if x.dtype not in (torch.float16, torch.bfloat16) or (dtype is not None and x.dtype != dtype) or x.device != like.device:
        raise ValueError(f"{name}: fp16 or bf16 on {like.device}, all alike; got {x.dtype} on {x.device}")


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
    kind, blocks, heads, bs, dim = _cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _rows(k, "k", heads, dim, k_cache)
    _rows(v, "v", heads, dim, k_cache, k.dtype)
    tokens = k.shape[0]
    _need(v.shape[0] == tokens, f"k has {tokens} tokens, v {v.shape[0]}")
    sl = _ints(slots, "slots", tokens, dev, torch.int64)
    qp = qo = fp = pp = None
    qt = qh = nq = limit = 0
    if freqs is not None:
        _need(positions is not None, "freqs needs positions")
        if freqs.dtype != torch.float32 or freqs.dim() != 3 or freqs.shape[1:] != (dim // 2, 2) or not freqs.is_contiguous() or freqs.device != dev:
            raise ValueError(f"freqs: contiguous fp32 [positions, {dim // 2}, 2] on {dev}, got {tuple(freqs.shape)} {freqs.dtype}")
        limit = freqs.shape[0]
        fp, pp = freqs.data_ptr(), _ints(positions, "positions", tokens, dev, torch.int64)
    if q is not None:
        _need(freqs is not None, "q is only rotated, which needs freqs")
        _rows(q, "q", None, dim, k_cache, k.dtype)
        _need(q.shape[0] == tokens, f"k has {tokens} tokens, q {q.shape[0]}")
        nq = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or not q_out.is_contiguous() or q_out.device != dev:
            raise ValueError("q_out: contiguous and like q")
        qp, qo, qt, qh = q.data_ptr(), q_out.data_ptr(), q.stride(0), q.stride(1)
    status = lib().gdsq_append_kv8(
        _ELEM[k.dtype], qp, qt, qh, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), qo,
        fp, limit, pp, sl, tokens, nq, heads, dim, kind, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), blocks, bs, torch.cuda.current_stream(dev).cuda_stream)
    if status:
        check(status, "gdsq_append_kv8")
    return q_out if q is not None else None


def attend_workspace(num_requests: int, max_query_len: int, num_heads: int, num_kv_heads: int, head_dim: int,
                     device) -> torch.Tensor:
    """A zeroed workspace for ``attend_kv8`` calls up to these sizes.  Keep it
    from call to call; calls that may run at the same time need one each."""
    n = lib().gdsq_attend_kv8_workspace(num_requests, max_query_len, num_heads, num_kv_heads, head_dim)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def attend_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, query_starts: torch.Tensor,
               max_query_len: int, max_seq_len: int | None = None, *, softmax_scale: float | None = None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens q [T, heads, dim] over the cache: request
    r's tokens are ``query_starts[r]:query_starts[r + 1]``, the last of its
    ``seq_lens[r]``, and each sees the positions up to its own.  Heads share KV
    heads in order (heads a multiple of kv_heads).  ``max_query_len`` and
    ``max_seq_len`` (default: what the block table can hold) bound the
    lengths, which the host does not see.  Returns [T, heads, dim]; a query
    that sees nothing gives zeros.  ``workspace``: see ``attend_workspace``
    (allocated for the call when not given)."""
    kind, blocks, heads, bs, dim = _cache(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _rows(q, "q", None, dim, k_cache)
    tokens, nq = q.shape[0], q.shape[1]
    r = seq_lens.numel()
    _need(block_table.dim() == 2 and block_table.shape[0] == r, f"block_table {tuple(block_table.shape)} has not {r} rows")
    width = block_table.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("out: contiguous and like q")
    if workspace is None:
        workspace = attend_workspace(r, max_query_len, nq, heads, dim, dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace: contiguous on {dev}")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(dim)
    status = lib().gdsq_attend_kv8(
        q.data_ptr(), _ELEM[q.dtype], q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), kind,
        k_scale.data_ptr(), v_scale.data_ptr(), blocks, bs, _ints(block_table, "block_table", r * width, dev), width,
        _ints(seq_lens, "seq_lens", r, dev), _ints(query_starts, "query_starts", r + 1, dev), r, tokens,
        max_query_len, width * bs if max_seq_len is None else max_seq_len, nq, heads, dim, softmax_scale,
        out.data_ptr(), workspace.data_ptr(), workspace.nbytes, torch.cuda.current_stream(dev).cuda_stream)
    if status:
        check(status, "gdsq_attend_kv8")
    return out
