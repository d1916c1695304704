"""Choosing the next tokens on the GPU.

GdsLLM samples on the host, one row at a time (gdsllm/engine.py:47-95).
``sample`` picks one token for every row of logits in one launch, from one
uniform number per row, with each row's own temperature, top-k, top-p and
min-p."""
from __future__ import annotations

import torch

from ._native import ext


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
    return ext().sample(logits, uniforms, temperature, top_k, top_p, min_p, tokens, logprobs)
