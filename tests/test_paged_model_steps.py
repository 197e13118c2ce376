"""Steps over a paged cache beside their results: the memory they take, what a refused one
leaves, and what they wait for."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from helpers import TINY, synth
from paged_helpers import sample_plain
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


class Busy:
    """Half a second of one thread's work on a stream; `running` afterwards: nothing waited for it."""

    def __init__(self, stream):
        import torch
        self.stream, self.done = stream, torch.cuda.Event()

    def __enter__(self):
        import torch
        torch.cuda.synchronize()
        with torch.cuda.stream(self.stream):
            torch.cuda._sleep(1_000_000_000)
            self.done.record()
        return self

    def __exit__(self, *_):
        self.stream.synchronize()

    def running(self):
        return not self.done.query()


@gpu
def test_sampled_steps_do_not_wait_for_other_streams(lib):
    import torch
    m = synth(lib, dict(TINY, n_layers=1), seed=14)
    kvs = [lib.q_llama_kv_create(C.byref(m)) for _ in range(2)]
    cache = lib.q_llama_paged_create(C.byref(m), 4, 16, 2, llmq.LLMQ_F32)
    llmq.check(lib)
    ids = llmq.int_array([-9, -9])
    s = llmq.sampling([0.8, 0.8], u=[0.3, 0.6])

    def steps():
        assert lib.q_llama_decode_batch_sample(C.byref(m), llmq.kv_pointers(kvs), llmq.int_array([5, 6]), 2, C.byref(s),
                                               ids) == 0
        step(lib, m, cache, [1, 1], [5, 6], 2, s)

    steps()
    with Busy(torch.cuda.Stream()) as busy:
        steps()
        assert busy.running()
    for kv in kvs:
        lib.llama_kv_free(C.byref(kv))
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_settings_follow_batches_that_grow_and_shrink(lib):
    """Batches of other sizes and columns one after another, each by its own settings."""
    m = synth(lib, dict(TINY, n_layers=1), seed=16, stddev=0.05)
    g = np.random.default_rng(4)
    cache = lib.q_llama_paged_create(C.byref(m), 70, 4, 70, llmq.LLMQ_F32)
    llmq.check(lib)
    for n in (2, 70, 1, 33):
        added = [1 if b < n else 0 for b in range(70)]
        u = g.random(70).astype(np.float32)
        cols = dict(top_k=g.integers(1, 50, 70)) if n % 2 else dict(temperature=g.choice([0.7, 1.3], 70), min_p=[0.01] * 70)
        ids, rows = step(lib, m, cache, added, g.integers(0, m.vocab, n).tolist(), 70, llmq.sampling(u=u, **cols))
        for b in range(n):
            want, _, margin = sample_plain(rows[b], float(np.float32(cols.get("temperature", [1.0] * 70)[b])),
                                           int(cols.get("top_k", [0] * 70)[b]), 1.0,
                                           float(np.float32(cols.get("min_p", [0.0] * 70)[b])), float(u[b]))
            assert margin < m.vocab * 2.0 ** -44 or ids[b] == want
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_steps_and_resets_do_not_wait_for_the_default_stream(lib):
    import torch
    m = synth(lib, dict(TINY, n_layers=1), seed=15)
    cache = lib.q_llama_paged_create(C.byref(m), 4, 16, 2, llmq.LLMQ_F32)
    llmq.check(lib)
    first, want = step(lib, m, cache, [5, 1], [1, 2, 3, 4, 5, 9], 2)
    with Busy(torch.cuda.default_stream()) as busy:
        assert lib.q_llama_paged_reset(cache, 0) == 0 and lib.q_llama_paged_reset(cache, 1) == 0
        ids, rows = step(lib, m, cache, [5, 1], [1, 2, 3, 4, 5, 9], 2)
        assert busy.running()
    assert ids == first and np.array_equal(rows.view(np.uint32), want.view(np.uint32))
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_launches_of_sampled_and_paged_steps(lib):
    """The sampler is one more kernel than the greedy step; over pages a layer has the writer,
    attention and its join in place of the writer, scores and values, and the step a plan and
    a copy of its last rows besides."""
    m = synth(lib, TINY, seed=17)
    kvs = [lib.q_llama_kv_create(C.byref(m)) for _ in range(2)]
    cache = lib.q_llama_paged_create(C.byref(m), 32, 16, 2, llmq.LLMQ_F32)
    llmq.check(lib)
    toks, ids = llmq.int_array([5, 6]), llmq.int_array([-9, -9])
    s = llmq.sampling([0.8, 0.8], u=[0.3, 0.6])
    assert lib.q_llama_decode_batch_argmax(C.byref(m), llmq.kv_pointers(kvs), toks, 2, ids) == 0
    greedy = lib.llmq_last_launches()
    assert lib.q_llama_decode_batch_sample(C.byref(m), llmq.kv_pointers(kvs), toks, 2, C.byref(s), ids) == 0
    assert lib.llmq_last_launches() == greedy + 1
    step(lib, m, cache, [1, 1], [5, 6], 2)
    assert lib.llmq_last_launches() == greedy + 2
    step(lib, m, cache, [1, 1], [5, 6], 2, s)
    assert lib.llmq_last_launches() == greedy + 3
    for kv in kvs:
        lib.llama_kv_free(C.byref(kv))
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))
