"""The batch path when something goes wrong in the middle of a step."""
from __future__ import annotations

import pytest
import torch

from gdsllm_b200 import batch, capi, paged
from test_batch_gpu import SHAPE, example

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda):
    return example.random_model(device=cuda, seed=1, max_seq=512, **SHAPE)


def served(model, cache):
    return batch.BatchLlama(*model, SHAPE["heads"], SHAPE["kv_heads"], 1e-5, max_requests=3, num_blocks=20, block_size=16, cache_dtype=cache)


@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("call", ["append_kv8", "attend_kv8"])
def test_a_step_that_raises_can_be_tried_again(cuda, model, monkeypatch, cache, call):
    """After an exception in the second layer the same step gives the same bits as where nothing went wrong."""
    steps = [[[1, 2, 3], list(range(40)), []], [[4], [5], [6, 7]], [[8] * 14, [9], []]]
    good, bad = served(model, cache), served(model, cache)
    for tokens in steps:
        want = good.step(tokens)
        state = (list(bad.lengths), bad.blocks_left, bad.free_head.item())
        calls, real = [], getattr(paged, call)

        def failing(*args, **kw):
            calls.append(0)
            if len(calls) == 2:
                raise RuntimeError("out of memory")
            return real(*args, **kw)

        monkeypatch.setattr(paged, call, failing)
        with pytest.raises(RuntimeError, match="out of memory"):
            bad.step(tokens)
        monkeypatch.setattr(paged, call, real)
        assert (list(bad.lengths), bad.blocks_left, bad.free_head.item()) == state
        got = bad.step(tokens)
        for r, t in enumerate(tokens):
            if t:
                assert torch.equal(got[r], want[r])
        assert bad.lengths == good.lengths and bad.blocks_left == good.blocks_left
    for r in range(3):
        bad.release(r)
    assert bad.blocks_left == 20 and sorted(bad.free.tolist()) == list(range(20))
    assert capi.device_error(0) == 0


def test_generate_no_tokens(cuda, model):
    b = served(model, torch.int8)
    tokens, logprobs = b.generate([[1, 2], [3]], 0)
    assert tokens.shape == logprobs.shape == (2, 0) and tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    assert b.blocks_left == 20 and b.lengths == [0, 0, 0]
    with pytest.raises(ValueError, match="-1 new tokens"):
        b.generate([[1, 2], [3]], -1)
