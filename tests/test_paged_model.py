"""A model's batches over a paged cache (q_llama_paged_*) and sampled batched decode:
against the single-sequence step, against the documented sampling rules on the logits
they return, and their refusals."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from helpers import TINY, gpu_decode, synth
from paged_helpers import sample_plain

gpu = pytest.mark.gpu


# ------------------------------------------------------------ refusals (CPU)
def refused(lib, code, fn, *args, result=None):
    lib.q_llama_clear_error()
    got = fn(*args)
    assert got == (code if result is None else result) or (result is None and got is None)
    assert lib.q_llama_last_error() == code
    lib.q_llama_clear_error()


def test_refusals_without_a_gpu(lib):
    m = llmq.QLlamaModel(head_dim=60)
    for n_pages, page, seqs, dtype in [(0, 16, 1, 0), (4, 0, 1, 0), (4, 16, 0, 0), (4, 16, 1, 3), (4, 16, 1, -1),
                                       (1 << 20, 1 << 12, 1, 0), (4, 16, 1, 0)]:  # the last: head_dim 60
        refused(lib, llmq.LLMQ_ERR_ARG, lambda: lib.q_llama_paged_create(C.byref(m), n_pages, page, seqs, dtype))
    one = llmq.int_array([1])
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_step, C.byref(m), 0x1000, one, one, None, one, None)
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_reset, 0x1000, 0)
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_len, 0x1000, 0, result=-1)
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_free_pages, None, result=-1)
    refused(lib, llmq.LLMQ_ERR_STATE, lambda: lib.q_llama_paged_free(0x1000))
    lib.q_llama_paged_free(None)
    s = llmq.sampling(u=[0.5])
    kv = llmq.kv_pointers([llmq.LlamaKV()])
    for args in [(kv, one, 0, C.byref(s), one), (kv, one, 1, None, one), (kv, one, 1, C.byref(s), None),
                 (kv, one, 1, C.byref(llmq.sampling(top_k=[1])), one)]:
        refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_decode_batch_sample, C.byref(m), *args)


def test_pages_that_attention_would_refuse(lib):
    m = llmq.QLlamaModel(head_dim=64)
    for n_pages, page in [(1, (1 << 31) - 4096), (1, (1 << 31) - 1), ((1 << 31) - 4000, 1)]:
        lib.q_llama_clear_error()
        assert lib.q_llama_paged_create(C.byref(m), n_pages, page, 1, llmq.LLMQ_BF16) is None
        assert b"bad sizes" in lib.q_llama_last_error_message()
    lib.q_llama_clear_error()


# ------------------------------------------------------------------- GPU
def step(lib, m, cache, added, tokens, seqs, s=None, want=True):
    n = sum(a > 0 for a in added)
    ids = llmq.int_array([-9] * seqs)
    rows = np.zeros((max(n, 1), m.vocab), np.float32)
    t = llmq.host_tensor(rows)
    rc = lib.q_llama_paged_step(C.byref(m), cache, llmq.int_array(added), llmq.int_array(tokens),
                                None if s is None else C.byref(s), ids, C.byref(t) if want else None)
    assert rc == 0, lib.q_llama_last_error_message()
    return list(ids), rows[:n]


def near(got, want, far):
    d = np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want.astype(np.float64))
    assert d <= far, d


# Attention differs from the reference's order by f32 roundings, about 1e-6 of itself.
# An activation within that of a rounding border takes the neighbouring int8 code, one
# 127th of its row's largest: some 3 roundings in 10^4, and each moves a product by about
# 0.3% of its norm.  2% leaves room for dozens.  16-bit pages round every key and value by
# up to 2^-9, which moves one code in ten: the bound is the reference's own for int8
# against f32 logits (selftest.c:1215-1250).
FAR = {llmq.LLMQ_F32: 0.02, llmq.LLMQ_F16: 0.15, llmq.LLMQ_BF16: 0.15}


@gpu
@pytest.mark.parametrize("dtype", [llmq.LLMQ_F32, llmq.LLMQ_F16, llmq.LLMQ_BF16])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_prompts_pieces_and_decode(lib, dtype, page):
    """Three of four sequences: a prompt at once, one in pieces, one that joins later; then
    decode steps, fed with the same ids as the single-sequence path."""
    m = synth(lib, TINY, seed=5, with_bias=True)
    g = np.random.default_rng(page)
    ids = [g.integers(0, m.vocab, n).tolist() for n in (21, 0, 40, 9)]
    ref = [gpu_decode(lib, m, x)[0] if x else None for x in ids]
    n_pages = sum(-(-len(x) // page) for x in ids) + 1
    cache = lib.q_llama_paged_create(C.byref(m), n_pages, page, 4, dtype)
    llmq.check(lib)
    at = [0, 0, 0, 0]
    for added in [[17, 0, 8, 0], [1, 0, 25, 0], [0, 0, 1, 7], [1, 0, 1, 1], [1, 0, 1, 1], [1, 0, 4, 0], [0, 0, 0, 0]]:
        tokens = [t for b, a in enumerate(added) for t in ids[b][at[b]:at[b] + a]]
        out, rows = step(lib, m, cache, added, tokens, 4)
        i = 0
        for b, a in enumerate(added):
            at[b] += a
            assert lib.q_llama_paged_len(cache, b) == at[b]
            if not a:
                assert out[b] == -1
                continue
            near(rows[i], ref[b][at[b] - 1], FAR[dtype])
            assert out[b] == int(np.argmax(rows[i]))
            i += 1
    assert at == [21, 0, 40, 9] and lib.q_llama_paged_free_pages(cache) == 1
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_prompts_of_several_passes(lib):
    """2300 rows in one step (three passes), the last rows of both sequences in different ones."""
    cfg = dict(TINY, max_seq=1500, n_layers=2)
    m = synth(lib, cfg, seed=6)
    g = np.random.default_rng(2)
    a, b = g.integers(0, m.vocab, 900).tolist(), g.integers(0, m.vocab, 1400).tolist()
    cache = lib.q_llama_paged_create(C.byref(m), 160, 16, 2, llmq.LLMQ_F32)
    llmq.check(lib)
    out, rows = step(lib, m, cache, [900, 1400], a + b, 2)
    for ids, row in ((a, rows[0]), (b, rows[1])):
        kv = lib.q_llama_kv_create(C.byref(m))
        want = np.zeros((1, m.vocab), np.float32)
        t = llmq.host_tensor(want)
        lib.q_llama_prefill(C.byref(m), C.byref(kv), llmq.int_array(ids), len(ids), C.byref(t))
        llmq.check(lib)
        near(row, want[0], 0.02)
        lib.llama_kv_free(C.byref(kv))
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_sampled_steps_follow_the_rules(lib):
    """The ids of a sampled step are what the rules give on the logits it returns; the same of
    q_llama_decode_batch_sample on q_llama_decode_batch's logits."""
    m = synth(lib, TINY, seed=7, stddev=0.05)
    g = np.random.default_rng(1)
    T, k = [0.8, 1.0, 0.0, 1.3, 0.7], [40, 0, 5, 300, 0]
    p, mp, u = [0.95, 1.0, 1.0, 0.9, 0.8], [0.0, 0.02, 0.0, 0.0, 0.0], g.random(5).astype(np.float32)
    s = llmq.sampling(T, k, p, mp, u)
    cache = lib.q_llama_paged_create(C.byref(m), 8, 16, 5, llmq.LLMQ_BF16)
    llmq.check(lib)
    f = [float(np.float32(x)) for x in T], [float(np.float32(x)) for x in p], [float(np.float32(x)) for x in mp]
    for added in ([3, 2, 0, 1, 4], [1, 1, 1, 1, 1]):
        tokens = g.integers(0, m.vocab, sum(added)).tolist()
        ids, rows = step(lib, m, cache, added, tokens, 5, s)
        act = [b for b in range(5) if added[b]]
        for row, b in zip(rows, act):
            want, _, margin = sample_plain(row, f[0][b], k[b], f[1][b], f[2][b], float(u[b]))
            assert margin < m.vocab * 2.0 ** -44 or ids[b] == want
    lib.q_llama_paged_free(cache)
    kvs = [lib.q_llama_kv_create(C.byref(m)) for _ in range(10)]
    logits = np.zeros((5, m.vocab), np.float32)
    t = llmq.host_tensor(logits)
    toks = llmq.int_array(g.integers(0, m.vocab, 5))
    lib.q_llama_decode_batch(C.byref(m), llmq.kv_pointers(kvs[:5]), toks, 5, C.byref(t))
    llmq.check(lib)
    ids = llmq.int_array([-9] * 5)
    assert lib.q_llama_decode_batch_sample(C.byref(m), llmq.kv_pointers(kvs[5:]), toks, 5, C.byref(s), ids) == 0
    for b in range(5):
        want, _, margin = sample_plain(logits[b], f[0][b], k[b], f[1][b], f[2][b], float(u[b]))
        assert margin < m.vocab * 2.0 ** -44 or ids[b] == want
        assert kvs[5 + b].len == 1
    for kv in kvs:
        lib.llama_kv_free(C.byref(kv))
    lib.q_llama_model_free(C.byref(m))


@gpu
def test_pages_run_out_come_back_and_serve_again(lib):
    m = synth(lib, dict(TINY, n_layers=2), seed=8)
    g = np.random.default_rng(3)
    x = g.integers(0, m.vocab, 30).tolist()
    cache = lib.q_llama_paged_create(C.byref(m), 5, 8, 3, llmq.LLMQ_F32)
    llmq.check(lib)
    first, _ = step(lib, m, cache, [16, 0, 16], x[:16] + x[:16], 3)
    assert first[0] == first[2] and lib.q_llama_paged_free_pages(cache) == 1
    one, rows = llmq.int_array([-9] * 3), None
    refused(lib, llmq.LLMQ_ERR_OOM, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([0, 9, 0]),
            llmq.int_array(x[:9]), None, one, None)
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([0, 41, 0]),
            llmq.int_array(x), None, one, None)  # more than all pages hold
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([0, -1, 0]),
            llmq.int_array(x), None, one, None)
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([0, 1, 0]),
            llmq.int_array([m.vocab]), None, one, None)
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_step, C.byref(m), cache, llmq.int_array([0, 1, 0]),
            None, None, one, None)
    refused(lib, llmq.LLMQ_ERR_ARG, lib.q_llama_paged_reset, cache, 3)
    assert [lib.q_llama_paged_len(cache, b) for b in range(3)] == [16, 0, 16]
    step(lib, m, cache, [0, 8, 0], x[:8], 3)  # the last free page
    assert lib.q_llama_paged_free_pages(cache) == 0
    assert lib.q_llama_paged_reset(cache, 0) == 0 and lib.q_llama_paged_free_pages(cache) == 2
    assert lib.q_llama_paged_reset(cache, 0) == 0
    _, want = step(lib, m, cache, [0, 8, 0], x[8:16], 3)  # sequence 1 goes on in a returned page
    ids, got = step(lib, m, cache, [0, 0, 0], [], 3)
    assert ids == [-1, -1, -1]
    ref, _ = gpu_decode(lib, m, x[:16])
    near(want[0], ref[15], 0.02)
    ids, rows = step(lib, m, cache, [8, 0, 0], x[:8], 3)
    near(rows[0], ref[7], 0.02)
    lib.q_llama_paged_free(cache)
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_len, cache, 0, result=-1)
    cache = lib.q_llama_paged_create(C.byref(m), 5, 8, 3, llmq.LLMQ_F32)
    lib.q_llama_model_free(C.byref(m))  # frees the cache
    refused(lib, llmq.LLMQ_ERR_STATE, lib.q_llama_paged_len, cache, 0, result=-1)


@gpu
def test_batched_decode_is_what_it_was(lib):
    """A greedy batched step beside a paged one gives the single-sequence logits, bit for bit."""
    m = synth(lib, TINY, seed=9)
    ids = [[5, 6, 7], [100, 3, 9]]
    ref = [gpu_decode(lib, m, x)[0] for x in ids]
    cache = lib.q_llama_paged_create(C.byref(m), 4, 16, 2, llmq.LLMQ_F32)
    kvs = [lib.q_llama_kv_create(C.byref(m)) for _ in range(2)]
    out = np.zeros((2, m.vocab), np.float32)
    t = llmq.host_tensor(out)
    for i in range(3):
        toks = llmq.int_array([x[i] for x in ids])
        step(lib, m, cache, [1, 1], list(toks), 2, want=False)
        lib.q_llama_decode_batch(C.byref(m), llmq.kv_pointers(kvs), toks, 2, C.byref(t))
        llmq.check(lib)
        for b in range(2):
            assert np.array_equal(out[b].view(np.uint32), ref[b][i].view(np.uint32))
    for kv in kvs:
        lib.llama_kv_free(C.byref(kv))
    lib.q_llama_paged_free(cache)
    lib.q_llama_model_free(C.byref(m))
