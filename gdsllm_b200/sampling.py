"""Choosing the next tokens on the GPU.

GdsLLM samples on the host, one row at a time (gdsllm/engine.py:47-95).
``sample`` picks one token for every row of logits in one launch, from one
uniform number per row, with each row's own temperature, top-k, top-p and
min-p."""
from __future__ import annotations

import torch

from ._native import check, lib
from .paged import _ELEM, _ints


def _param(t: torch.Tensor | None, name: str, rows: int, device, dtype=torch.float32) -> int | None:
    return None if t is None else _ints(t, name, rows, device, dtype)


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           tokens: torch.Tensor | None = None, logprobs: torch.Tensor | None = None):
    """(tokens int64 [B], logprobs fp32 [B]) for logits [B, V] (fp16, bf16 or
    fp32; V up to 524288, contiguous rows) and ``uniforms`` fp32 [B] in [0, 1).

    Per row: weights floor(2^31 exp((l - max) / temperature)), whole numbers;
    then the longest prefix, by falling logit (ties: lowest index first),
    inside the ``top_k`` largest, with less than ``top_p`` of their weight
    before each, and with probability at least ``min_p`` times the largest's.
    The token is the first kept index whose running weight exceeds
    floor(uniform * kept weight), and its log-probability is that of its
    share.  Temperature 0 takes the largest logit.  Each parameter is a [B]
    tensor (top_k int32, the rest fp32) or None.  A row with no logit above
    -inf gives token -1; NaN counts as -inf."""
    if logits.dim() != 2 or logits.dtype not in _ELEM or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits: [rows, vocab] fp16, bf16 or fp32 with contiguous rows, got {tuple(logits.shape)} "
                         f"{logits.dtype} strides {logits.stride()}")
    b, v = logits.shape
    dev = logits.device
    if tokens is None:
        tokens = torch.empty(b, dtype=torch.int64, device=dev)
    if logprobs is None:
        logprobs = torch.empty(b, dtype=torch.float32, device=dev)
    status = lib().gdsq_sample(
        _ELEM[logits.dtype], logits.data_ptr(), logits.stride(0), b, v, _ints(uniforms, "uniforms", b, dev, torch.float32),
        _param(temperature, "temperature", b, dev), _param(top_k, "top_k", b, dev, torch.int32),
        _param(top_p, "top_p", b, dev), _param(min_p, "min_p", b, dev), _ints(tokens, "tokens", b, dev, torch.int64),
        _ints(logprobs, "logprobs", b, dev, torch.float32), torch.cuda.current_stream(dev).cuda_stream)
    if status:
        check(status, "gdsq_sample")
    return tokens, logprobs
