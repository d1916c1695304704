"""More of what the batched-serving entry points refuse, without a GPU."""
from __future__ import annotations

import pytest

from gdsllm_b200._native import lib

P = 0x100000  # never dereferenced
NAMES = ["context_lens", "new_lens", "block_table", "free_blocks", "free_head", "seq_lens", "query_starts", "positions", "slots", "free_head_out"]
REQUESTS, WIDTH, FREE, TOKENS = 5, 3, 7, 9
BYTES = dict(context_lens=4 * REQUESTS, new_lens=4 * REQUESTS, block_table=4 * REQUESTS * WIDTH, free_blocks=4 * FREE, free_head=4, seq_lens=4 * REQUESTS,
             query_starts=4 * (REQUESTS + 1), positions=8 * TOKENS, slots=8 * TOKENS, free_head_out=4)


def tables(**moved):
    at = {n: P + 0x1000 * i for i, n in enumerate(NAMES)}
    at.update(moved)
    return lib().gdsq_build_tables(at["context_lens"], at["new_lens"], REQUESTS, at["block_table"], WIDTH, at["free_blocks"], FREE, at["free_head"],
                                   16, TOKENS, at["seq_lens"], at["query_starts"], at["positions"], at["slots"], at["free_head_out"], None)


@pytest.mark.parametrize("output", ["seq_lens", "query_starts", "positions", "slots", "free_head_out", "block_table"])
def test_tables_refuse_an_output_that_overlaps(output):
    """The same address, the output's last word on the other's first, and the other way round (8-byte steps where alignment asks for them)."""
    step = 8 if output in ("positions", "slots") else 4
    for other in NAMES:
        if other == output:
            continue
        base = P + 0x1000 * NAMES.index(other)
        for at in (base, base - BYTES[output] + step, base + BYTES[other] // step * step - (0 if BYTES[other] % step else step)):
            assert tables(**{output: at}) == 1, (output, other, at)
            text = lib().gdsq_last_error()
            assert (b"overlaps" in text or b"must not be" in text) and output.encode() in text, text


def attend(width, block, requests=1):
    return lib().gdsq_attend_kv8(P, 0, 64, 64, P, P, 0, P, P, 4, block, P, width, P, P, requests, 1, 1, 64, 2, 1, 64, 0.1, P, P, 1 << 30, None)


@pytest.mark.parametrize("width,block", [(1 << 27, 16), (1 << 24, 128), ((1 << 26) - 1, 32), (2 ** 31 - 1, 64)])
def test_attend_refuses_a_table_row_past_31_bits(width, block):
    """table_width * block_size is a position in the kernels."""
    assert attend(width, block) == 3
    assert b"positions" in lib().gdsq_last_error()
