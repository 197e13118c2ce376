"""llmq_sample_rows: a token for each row of logits from given random numbers,
against the documented rules in 64 bits, against sample_token, and its
refusals (which need no GPU)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from conftest import has_gpu
from helpers import sampler_rows
from paged_helpers import CODES, ok, ptr, sample_gpu, sample_plain, torch_type

gpu = pytest.mark.gpu
F = 0x10000


def args(**kw):
    d = dict(n_rows=2, vocab=100, dtype=0, logits=F, stride=100, u=F, ids=F)
    d.update(kw)
    return llmq.SampleRows(**d)


@pytest.mark.parametrize("bad", [dict(n_rows=-1), dict(vocab=0), dict(vocab=-4), dict(vocab=(1 << 20) + 1, stride=1 << 22),
                                 dict(dtype=3), dict(logits=None), dict(u=None), dict(ids=None), dict(stride=99),
                                 dict(logits=F + 2), dict(dtype=1, logits=F + 1)], ids=str)
def test_refuses(lib, bad):
    lib.q_llama_clear_error()
    assert lib.llmq_sample_rows(C.byref(args(**bad)), None) == llmq.LLMQ_ERR_ARG == lib.q_llama_last_error()
    assert lib.q_llama_last_error_message().startswith(b"llmq_sample_rows")
    lib.q_llama_clear_error()


def test_null_and_empty(lib):
    assert lib.llmq_sample_rows(None, None) == llmq.LLMQ_ERR_ARG
    lib.q_llama_clear_error()
    assert lib.llmq_sample_rows(C.byref(args(n_rows=0)), None) == 0


@pytest.mark.skipif(has_gpu(), reason="this machine has a GPU")
def test_good_call_without_a_gpu_says_so(lib):
    assert lib.llmq_sample_rows(C.byref(args()), None) == llmq.LLMQ_ERR_NO_DEVICE
    lib.q_llama_clear_error()


def test_plain_rules_by_hand():
    row = [0.0, np.log(4.0), np.log(4.0), -np.inf, np.log(2.0), np.nan]
    w = [4, 4, 2, 1]  # ids 1, 2, 4, 0
    assert [sample_plain(row, 1.0, 0, 1.0, 0, u)[0] for u in (0, 0.36, 0.37, 8.1 / 11, 10.1 / 11, 1)] == [1, 1, 2, 4, 0, 0]
    assert sample_plain(row, 1.0, 2, 1.0, 0, 1.0)[0] == 2
    assert sample_plain(row, 1.0, 0, 0.5, 0, 1.0)[0] == 2
    assert sample_plain(row, 1.0, 0, 1.0, 0.45, 1.0)[0] == 4
    assert sample_plain(row, 0.0, 0, 1.0, 0, 1.0)[:2] == (1, 0.0)
    assert abs(sample_plain(row, 1.0, 3, 1.0, 0, 1.0)[1] - np.log(w[2] / 10)) < 1e-12


SETTINGS = [(0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (1.3, 1000, 0.99, 0.001),
            (0.0, 40, 0.95, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 5, 0.3, 0.2), (2.0, 2000, 1.0, 0.0), (1.0, 0, 1e-9, 0.0),
            (0.05, 0, 0.999, 0.0), (1.0, 0, 1.0, 1.0), (float("nan"), 3, 0.5, 0.0), (-1.0, 0, 1.0, 0.0),
            (1.0, 10**9, 2.0, 7.0), (1.0, -5, -1.0, -1.0), (float("inf"), 0, 0.5, 0.0), (1e-30, 3, 0.5, 0.0),
            (30.0, 0, 0.99999, 0.0), (30.0, 30000, 0.9, 0.9)]
U = [0.0, 0.031, 0.5, 0.77, 0.9999, 0.99999994, 1.0]


def check_rows(lib, rows, dtype, settings, us, seed=0):
    """Every row with every setting and u, in one call a row set.  A weight is off by
    half of 2^-45 (its rounding to an integer, vocab <= 2^17) and 2^-46 of itself
    (its exponential), so a sum of V of them moves by at most V 2^-45 against a
    whole of at least 1; where a plain border is nearer than that to a choice, either
    neighbour is right and the row is left out.  The share's log: 2^-45 of it and an
    f32 rounding."""
    import torch
    t = torch.tensor(np.asarray(rows, np.float32)).to(torch_type(dtype))
    seen = t.double().numpy()
    combos = [(r, s, u) for r in range(len(rows)) for s in settings for u in us]
    x = t[[c[0] for c in combos]].cuda()
    cols = list(zip(*[c[1] for c in combos]))
    ids, lp = sample_gpu(lib, x, dtype, cols[0], cols[1], cols[2], cols[3], [c[2] for c in combos])
    checked = 0
    for (r, s, u), i, l in zip(combos, ids, lp):
        s = tuple(float(np.float32(v)) if n != 1 else v for n, v in enumerate(s))
        want, wl, margin = sample_plain(seen[r], *s, float(np.float32(u)))
        if margin < len(seen[r]) * 2.0 ** -44:
            continue
        checked += 1
        assert i == want, (r, s, u, i, want, margin)
        assert (np.isneginf(l) and np.isneginf(wl)) or abs(l - wl) <= 2.0 ** -23 * (1 + abs(wl)) + len(seen[r]) * 2.0 ** -43, (r, s, u, l, wl)
    assert checked >= 0.7 * len(combos)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 31, 32, 33, 1000, 1025, 4099])
def test_small_vocabularies(lib, V, dtype):
    g = np.random.default_rng(V)
    rows = [g.normal(0, 2, V), np.zeros(V), np.round(g.normal(0, 2, V)), g.normal(0, 30, V)]
    check_rows(lib, rows, dtype, SETTINGS, U)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [32000, 50257, 128256])
def test_large_vocabularies(lib, V, dtype):
    g = np.random.default_rng(V)
    x = g.normal(0, 2, V)
    y = x.copy()
    y[g.integers(0, V, 30)] += 9
    check_rows(lib, [x, y], dtype, SETTINGS, U[1:5])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_awkward_rows(lib, dtype):
    """Ties of whole rows, few distinct values, one word far above, a heavy tail, signed
    zeros, infinities, NaN, the type's lowest value, and nothing at all."""
    g = np.random.default_rng(9)
    V, big = 20000, np.finfo(np.float32).max
    two = np.where(g.random(V) < 0.5, 1.0, -1.0)
    spike = g.normal(0, 1, V)
    spike[777] = 60
    zeros = np.where(g.random(V) < 0.5, 0.0, -0.0)
    masked = np.full(V, -np.inf)
    masked[[5, 19999, 300]] = [1.0, 2.0, 2.0]
    lowest = np.full(V, -big)
    lowest[[8, 9]] = [0.5, 0.25]
    pinf = g.normal(0, 1, V)
    pinf[[4, 100, 9000]] = np.inf
    nan = g.normal(0, 1, V)
    nan[::3] = np.nan
    ramp = np.arange(V) * -1e-3
    rows = [np.full(V, 3.0), two, spike, zeros, masked, lowest, pinf, nan, np.full(V, -np.inf), np.full(V, np.nan),
            np.full(V, -big), ramp, ramp[::-1], np.where(np.arange(V) < 5000, 0.0, g.normal(-1, 0.1, V)),
            np.full(V, big), g.standard_cauchy(V)]
    check_rows(lib, rows, dtype, SETTINGS, U)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_min_p_without_top_p(lib, dtype):
    """What min_p asks for can be bounded beforehand: rows whose bound lies above zero, at
    it and below it, with NaN, infinities and the type's lowest value among them."""
    g = np.random.default_rng(12)
    V, big = 9001, np.finfo(np.float32).max
    x = g.normal(0, 2, V)
    holes = x + 6
    holes[::5], holes[1::5], holes[2::5] = np.nan, -np.inf, -big
    zero = np.where(g.random(V) < 0.5, x, 0.0)
    zero[zero > 0] = 0.0
    zero[[3, 8000]] = np.log(20.0)  # with min_p 0.05 the bound is next to 0
    tiny = g.normal(0, 1e-7, V)
    tiny[11] = 1e-6
    pinf = x.copy()
    pinf[[70, 4]] = np.inf
    rows = [x + 10, x - 10, x, holes, zero, tiny, tiny - 1, pinf, np.full(V, 7.0), np.full(V, -7.0), 40 * x]
    settings = [(1.0, 0, 1.0, 0.05), (1.0, 20, 1.0, 0.05), (1.0, 3000, 0.0, 0.001), (0.5, 0, 1.0, 1e-30),
                (3.0, 50, 0.0, 0.3), (float("inf"), 0, 1.0, 1.0), (float("inf"), 7, 1.0, 0.5), (1.0, 0, 1.0, 1.0),
                (0.01, 2, 1.0, 0.5), (20.0, 0, 1.0, 0.9)]
    check_rows(lib, rows, dtype, settings, U)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_of_tiny_logits(lib, dtype):
    """Logits of magnitudes far below the row's largest, on both sides of zero and with
    zeros among them: a histogram of values holds them together."""
    g = np.random.default_rng(10)
    V = 5000
    tiny = g.normal(0, 1e-6, V)
    one = tiny.copy()
    one[[17, 4000]] = 1.0
    neg = tiny.copy()
    neg[g.random(V) < 0.3] = -3.0
    zeros = np.where(g.random(V) < 0.5, tiny, 0.0)
    zeros[5] = 2.0
    few = np.full(V, -5.0)
    few[100:140] = np.linspace(-1e-5, 1e-5, 40)
    few[7] = 0.5
    spread = np.sign(g.normal(0, 1, V)) * 2.0 ** g.uniform(-40, 3, V)
    check_rows(lib, [tiny, one, neg, zeros, few, spread], dtype, SETTINGS, U + [0.2, 0.35, 0.65])


@gpu
def test_ties_go_to_the_lowest_index_exactly(lib):
    """V equal logits: u * kept falls on token ceil(u * kept) - 1, exactly."""
    import torch
    for V in (2, 3, 1000, 4096, 70001):
        x = torch.full((1, V), 1.5, device="cuda").expand(6, V).contiguous()
        us = [0.0, 0.25, 0.5, 0.75, 1.0, 0.999]
        k = [0, 0, 0, 3 if V > 3 else 0, 0, 0]
        ids, _ = sample_gpu(lib, x, "f32", 1.0, k, 1.0, 0.0, us)
        kept = [V, V, V, min(V, k[3] or V), V, V]
        want = [max(int(np.ceil(float(np.float32(u)) * n)) - 1, 0) for u, n in zip(us, kept)]
        assert ids.tolist() == want, V
        ids, _ = sample_gpu(lib, x, "f32", 0.0, u=us)
        assert ids.tolist() == [0] * 6


@gpu
def test_optional_columns_and_u_outside(lib):
    import torch
    x = torch.tensor(np.random.default_rng(3).normal(0, 2, (4, 999)), dtype=torch.float32, device="cuda")
    ids, _ = sample_gpu(lib, x, "f32", u=[float("nan"), -3.0, 1.5, float("inf")], want=False)
    row = x.double().cpu().numpy()
    assert ids[0] == row[0].argmax() and ids[1] == row[1].argmax()
    assert ids[2] == row[2].argmin() and ids[3] == row[3].argmin()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("V,pad,lead", [(1000, 3, 0), (1000, 0, 1), (33, 7, 5), (128256, 1, 3)])
def test_strides_and_starts(lib, V, pad, lead, dtype):
    import torch
    g = np.random.default_rng(V + pad)
    raw = torch.tensor(g.normal(0, 2, 5 * (V + pad) + lead), dtype=torch_type(dtype), device="cuda")
    x = raw[lead:].view(5, V + pad)[:, :V]
    s = (0.9, 50, 0.9, 0.01)
    ids, _ = sample_gpu(lib, x, dtype, *s, u=[0.1, 0.3, 0.5, 0.7, 0.9])
    same, _ = sample_gpu(lib, x.contiguous(), dtype, *s, u=[0.1, 0.3, 0.5, 0.7, 0.9])
    assert ids.tolist() == same.tolist()
    for r, u in enumerate([0.1, 0.3, 0.5, 0.7, 0.9]):
        want = sample_plain(x[r].double().cpu().numpy(), float(np.float32(0.9)), 50, 0.9, float(np.float32(0.01)),
                            float(np.float32(u)))
        assert want[2] < V * 2.0 ** -44 or ids[r] == want[0]


@gpu
def test_a_row_does_not_depend_on_its_batch(lib):
    """The same rows alone, in a small and in a large batch, on another stream, captured and
    replayed: the same ids and shares, bit for bit."""
    import torch
    g = np.random.default_rng(11)
    x = torch.tensor(g.normal(0, 2, (300, 40000)), dtype=torch.float32, device="cuda")
    T, k, p, mp = g.choice([0.7, 1.0, 1.4], 300), g.choice([0, 50, 1500], 300), g.choice([1.0, 0.9], 300), g.choice([0.0, 0.02], 300)
    u = g.random(300)
    ids, lp = sample_gpu(lib, x, "f32", T, k, p, mp, u)
    for lo, hi in ((0, 1), (7, 8), (100, 108), (40, 120)):
        i, l = sample_gpu(lib, x[lo:hi], "f32", T[lo:hi], k[lo:hi], p[lo:hi], mp[lo:hi], u[lo:hi],
                          stream=torch.cuda.Stream())
        assert (i == ids[lo:hi]).all() and (l.view(np.uint32) == lp[lo:hi].view(np.uint32)).all()
    f = dict(dtype=torch.float32, device="cuda")
    c = [torch.tensor(T, **f), torch.tensor(k, dtype=torch.int32, device="cuda"), torch.tensor(p, **f),
         torch.tensor(mp, **f), torch.tensor(u, **f)]
    out = torch.zeros(300, dtype=torch.int32, device="cuda")
    a = llmq.SampleRows(n_rows=300, vocab=40000, dtype=0, logits=ptr(x), stride=40000, temperature=ptr(c[0]),
                        top_k=ptr(c[1]), top_p=ptr(c[2]), min_p=ptr(c[3]), u=ptr(c[4]), ids=ptr(out))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok(lib, lib.llmq_sample_rows(C.byref(a), torch.cuda.current_stream().cuda_stream))
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (out.cpu().numpy() == ids).all()


@gpu
def test_calls_of_several_threads_at_once(lib):
    """Rows of different sizes and types, so that the calls' shared memory differs."""
    import threading

    import torch
    g = np.random.default_rng(21)
    jobs = [(V, t, torch.tensor(g.normal(0, 2, (3, V)), dtype=torch_type(t), device="cuda"))
            for V, t in ((500, "f32"), (128256, "f32"), (40000, "f32"), (9000, "bf16"), (128256, "bf16"))]
    s, u = (1.0, 0, 0.9, 0.0), [0.2, 0.5, 0.8]
    want = [sample_gpu(lib, x, t, *s, u=u)[0].tolist() for _, t, x in jobs]
    bad = []

    def work(i):
        f = dict(dtype=torch.float32, device="cuda")
        _, t, x = jobs[i]
        c = [torch.full((3,), v, **f) for v in (s[0], s[2])] + [torch.tensor(u, **f)]
        ids = torch.zeros(3, dtype=torch.int32, device="cuda")
        a = llmq.SampleRows(n_rows=3, vocab=x.shape[1], dtype=CODES[t], logits=ptr(x), stride=x.stride(0),
                            temperature=ptr(c[0]), top_p=ptr(c[1]), u=ptr(c[2]), ids=ptr(ids))
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(50):
            if lib.llmq_sample_rows(C.byref(a), st.cuda_stream) != 0:
                bad.append("error")
        st.synchronize()
        if ids.tolist() != want[i]:
            bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [300000, 1 << 20])
def test_largest_vocabularies(lib, V, dtype):
    import torch
    g = np.random.default_rng(V)
    x = torch.tensor(g.normal(0, 2, (1, V)), dtype=torch.float32).to(torch_type(dtype))
    x[0, V - 1] = 11.0
    row = x[0].double().numpy()
    for s in [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.7, 0.0), (1.0, 5000, 1.0, 0.0), (0.0, 0, 1.0, 0.0)]:
        for u in (0.0, 0.4, 0.97):
            i, _ = sample_gpu(lib, x.cuda(), dtype, *s, u=u)
            want, _, margin = sample_plain(row, *[float(np.float32(v)) if n != 1 else v for n, v in enumerate(s)],
                                           float(np.float32(u)))
            assert margin < V * 2.0 ** -41 or i[0] == want, (s, u)


@gpu
def test_agrees_with_sample_token(lib):
    """The rows and settings of sample_token's own tests, with the u its stream gives:
    the same token wherever f32 sums cannot move the choice."""
    import torch
    agreed = 0
    for name, row in sampler_rows().items():
        if np.isnan(row).any() or np.isposinf(row).any():
            continue  # the reference's NaN sums are its own
        for T, k, p in [(0.8, 40, 0.95), (0.9, 40, 0.95), (1.0, 1, 1.0), (1.5, 1000, 0.5), (0.0, 40, 0.95)]:
            rng, us, toks = llmq.Rng(77), [], []
            t = llmq.host_tensor(row.reshape(1, -1))
            for _ in range(6):
                probe = llmq.Rng(rng.state)
                us.append(lib.rng_uniform(C.byref(probe)))
                toks.append(lib.sample_token(C.byref(t), 0, T, k, p, C.byref(rng)))
                llmq.check(lib)
            x = torch.tensor(row, device="cuda").expand(6, -1).contiguous()
            ids, _ = sample_gpu(lib, x, "f32", T, k, p, 0.0, us)
            for i, tok, u in zip(ids, toks, us):
                margin = sample_plain(row, float(np.float32(T)), k, float(np.float32(p)), 0.0, u)[2]
                if margin > 1e-3:  # sequential f32 sums of up to 128256 terms
                    assert i == tok, (name, T, k, p, u)
                    agreed += 1
    assert agreed > 100


@gpu
def test_host_memory_is_refused(lib):
    import torch
    x, u, ids = torch.zeros((2, 10), device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in ("logits", "u", "ids"):
        d = dict(logits=x, u=u, ids=ids)
        d[bad] = d[bad].cpu()
        a = args(vocab=10, stride=10, **{n: ptr(t) for n, t in d.items()})
        assert lib.llmq_sample_rows(C.byref(a), None) == llmq.LLMQ_ERR_ARG
    lib.q_llama_clear_error()
