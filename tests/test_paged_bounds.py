"""Sharper forms of two checks of the paged cache: what a plan leaves of lengths out of range,
to the entry, and how near 16-bit pages of f16 keep a model's logits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from helpers import TINY, gpu_decode, synth
from paged_helpers import plan_gpu
from test_paged_model import FAR, near, step

gpu = pytest.mark.gpu


@gpu
def test_lengths_out_of_range_to_the_entry(lib):
    """48 positions a row: requests below 0, past the row, at its end, and three that are good,
    of which one lacks a page in its table."""
    table = np.full((8, 6), -1)
    table[4, :2] = [3, 4]
    table[5] = [5, 6, 7, 8, 9, 10]
    got = plan_gpu(lib, [-1, 3, 49, 48, 10, 47, 2**31 - 1, 20], [1, -2, 0, 1, 39, 1, 2**31 - 1, 3], 8, 6, 64,
                   [20, 21, 22, 23], 0, table)
    assert got["lens"].tolist() == [0, 3, 0, 48, 10, 48, 0, 23]
    assert got["first"].tolist() == [0, 0, 0, 0, 0, 0, 1, 1, 4]
    assert got["slots"].tolist() == [87, -1, -1, -1] + [-1] * 60
    assert got["positions"].tolist()[:5] == [47, 20, 21, 22, -1]
    assert got["status"] == llmq.LLMQ_PAGED_BAD_LEN | llmq.LLMQ_PAGED_BAD_PAGE and got["next_head"] == 0


# A key or value rounded to f16 is off by 2^-11 of itself at most, to bf16 by 2^-8: an eighth.
# The share of activations that a rounding moves to the neighbouring int8 code goes with
# its size, and the moves' sum, of either sign, with the root of their number.
F16_FAR = FAR[llmq.LLMQ_BF16] / 8 ** 0.5


@gpu
@pytest.mark.parametrize("page", [5, 16])
def test_f16_pages_are_nearer_than_bf16_ones(lib, page):
    m = synth(lib, TINY, seed=5, with_bias=True)
    ids = np.random.default_rng(page).integers(0, m.vocab, 44).tolist()
    ref = gpu_decode(lib, m, ids)[0]
    cache = lib.q_llama_paged_create(C.byref(m), -(-44 // page), page, 1, llmq.LLMQ_F16)
    llmq.check(lib)
    at = 0
    for n in (17, 1, 1, 20, 1, 4):
        _, rows = step(lib, m, cache, [n], ids[at:at + n], 1)
        at += n
        near(rows[0], ref[at - 1], F16_FAR)
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))
