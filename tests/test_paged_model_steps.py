"""Steps over a paged cache beside their results: the memory they take, what a refused one
leaves, and what they wait for."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from helpers import TINY, synth
from test_paged_model import refused, step

gpu = pytest.mark.gpu


@gpu
def test_a_step_takes_no_memory_for_contiguous_attention(lib):
    """500 rows at max_seq 36000: the contiguous path's scores would take 430 MB, the rows
    themselves 5 MB."""
    import torch
    m = synth(lib, dict(TINY, max_seq=36000, n_layers=1), seed=11)
    cache = lib.q_llama_paged_create(C.byref(m), 40, 16, 2, llmq.LLMQ_BF16)
    llmq.check(lib)
    tokens = np.random.default_rng(5).integers(0, m.vocab, 500).tolist()
    step(lib, m, cache, [1, 1], tokens[:2], 2)  # what any step needs once
    before = torch.cuda.mem_get_info()[0]
    step(lib, m, cache, [500, 0], tokens, 2)
    assert before - torch.cuda.mem_get_info()[0] < 100 << 20
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_a_pool_that_does_not_fit_is_out_of_memory(lib):
    """One page of 2^31 - 8192 positions of 96 floats: some 800 GB, refused by the allocator
    at once.  A smaller cache and its steps work afterwards."""
    m = synth(lib, dict(TINY, n_layers=1), seed=12)
    refused(lib, llmq.LLMQ_ERR_OOM, lambda: lib.q_llama_paged_create(C.byref(m), 1, (1 << 31) - 8192, 1, llmq.LLMQ_F32))
    cache = lib.q_llama_paged_create(C.byref(m), 2, 16, 1, llmq.LLMQ_F32)
    llmq.check(lib)
    step(lib, m, cache, [3], [1, 2, 3], 1)
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_a_step_the_sampler_would_refuse_is_refused_before_it_runs(lib):
    """A vocabulary past the sampler's limit: sampled steps are refused and leave the sequences
    as they were; greedy ones go on."""
    cfg = dict(TINY, vocab=(1 << 20) + 1, n_layers=1, d_model=96, n_heads=2, n_kv=1, d_ff=96, max_seq=64)
    m = synth(lib, cfg, seed=13)
    cache = lib.q_llama_paged_create(C.byref(m), 4, 16, 2, llmq.LLMQ_F32)
    llmq.check(lib)
    step(lib, m, cache, [3, 0], [1, 2, 3], 2, want=False)
    s = llmq.sampling(u=[0.5, 0.5])
    ids = llmq.int_array([-9, -9])
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([1, 20]),
            llmq.int_array(list(range(21))), C.byref(s), ids, None)
    assert lib.q_llama_paged_len(cache, 0) == 3 and lib.q_llama_paged_len(cache, 1) == 0
    assert lib.q_llama_paged_free_pages(cache) == 3
    step(lib, m, cache, [1, 20], list(range(21)), 2, want=False)
    assert lib.q_llama_paged_len(cache, 0) == 4 and lib.q_llama_paged_free_pages(cache) == 1
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))
