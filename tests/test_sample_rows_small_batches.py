"""llmq_sample_rows in small batches, whose rows are shared by clusters of up to eight CTAs:
ties across slices, infinities, NaN, tiny logits, bounds and rows that start anywhere give
the ids and shares of the large batch, a CTA a row, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from paged_helpers import sample_gpu, sample_plain, torch_type
from test_sample_rows import SETTINGS

gpu = pytest.mark.gpu
V = 20011  # clusters of eight in every type; slices that end inside a vector
U = [0.0, 0.031, 0.5, 0.9999, 1.0]


def awkward(g):
    big = np.finfo(np.float32).max
    two = np.where(g.random(V) < 0.5, 1.0, -1.0)
    late = np.full(V, -4.0)
    late[V - 9:] = 2.0  # ties in the last slice alone
    early = np.full(V, -4.0)
    early[[0, 1, 2501, 2502, 17500, V - 1]] = 0.25
    zeros = np.where(g.random(V) < 0.5, 0.0, -0.0)
    masked = np.full(V, -np.inf)
    masked[[5, V - 2, 300]] = [1.0, 2.0, 2.0]
    lowest = np.full(V, -big)
    lowest[[8, 19000]] = [0.5, 0.25]
    pinf = g.normal(0, 1, V)
    pinf[[4, 9000, V - 1]] = np.inf
    nan = g.normal(0, 1, V)
    nan[::3] = np.nan
    return [np.full(V, 3.0), two, late, early, zeros, masked, lowest, pinf, nan, np.full(V, -np.inf),
            np.full(V, np.nan), np.arange(V) * -1e-3, g.standard_cauchy(V)]


def tiny(g):
    small = g.normal(0, 1e-6, V)
    one = small.copy()
    one[[17, 14000]] = 1.0
    neg = small.copy()
    neg[g.random(V) < 0.3] = -3.0
    zeros = np.where(g.random(V) < 0.5, small, 0.0)
    zeros[5] = 2.0
    few = np.full(V, -5.0)
    few[100:V:500] = np.linspace(-1e-5, 1e-5, len(few[100:V:500]))
    few[7] = 0.5
    return [small, one, neg, zeros, few, np.sign(g.normal(0, 1, V)) * 2.0 ** g.uniform(-40, 3, V)]


def bounded(g):
    x = g.normal(0, 2, V)
    holes = x + 6
    holes[::5], holes[1::5] = np.nan, -np.inf
    zero = np.where(g.random(V) < 0.5, x, 0.0)
    zero[zero > 0] = 0.0
    zero[[3, 18000]] = np.log(20.0)
    return [x + 10, x - 10, x, holes, zero, np.full(V, 7.0), 40 * x]


BOUNDS = [(1.0, 0, 1.0, 0.05), (1.0, 20, 1.0, 0.05), (1.0, 3000, 0.0, 0.001), (0.5, 0, 1.0, 1e-30),
          (3.0, 50, 0.0, 0.3), (float("inf"), 0, 1.0, 1.0), (0.01, 2, 1.0, 0.5), (20.0, 0, 1.0, 0.9)]
SETS = {"awkward": (awkward, SETTINGS[:16]), "tiny": (tiny, SETTINGS[:16:2]), "bounded": (bounded, BOUNDS)}


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", SETS)
def test_small_batches_are_the_large_one(lib, name, dtype):
    import torch
    make, settings = SETS[name]
    t = torch.tensor(np.stack(make(np.random.default_rng(33))).astype(np.float32)).to(torch_type(dtype))
    seen = t.double().numpy()
    combos = [(r, s, u) for s in settings for u in U for r in range(len(t))]
    # rows that start on any element, their ends beside one another
    raw = torch.zeros(len(t) * (V + 3) + 1, dtype=t.dtype, device="cuda")
    rows = raw[1:].view(len(t), V + 3)[:, :V]
    rows.copy_(t)
    cols = [np.array([c[1][i] for c in combos], np.float64 if i != 1 else np.int64) for i in range(4)]
    us = np.array([c[2] for c in combos])
    large = t.cuda()[[c[0] for c in combos]]
    ids, lp = sample_gpu(lib, large, dtype, *cols, us)
    n = len(t)
    checked = 0
    for at in range(0, len(combos), n):  # a setting and a u: every row once
        for lo in range(0, n, 7):
            sl = slice(at + lo, at + min(n, lo + 7))
            i, l = sample_gpu(lib, rows[lo:min(n, lo + 7)], dtype, *[c[sl] for c in cols], us[sl])
            assert (i == ids[sl]).all(), (combos[sl], i, ids[sl])
            assert (l.view(np.uint32) == lp[sl].view(np.uint32)).all(), combos[sl]
    for (r, s, u), i in list(zip(combos, ids))[::11]:  # (the large batch has tests of its own)
        s = tuple(float(np.float32(v)) if k != 1 else v for k, v in enumerate(s))
        want, _, margin = sample_plain(seen[r], *s, float(np.float32(u)))
        if margin >= V * 2.0 ** -44:
            assert i == want, (r, s, u)
            checked += 1
    assert checked > len(combos) // 11 // 2


@gpu
@pytest.mark.parametrize("V,pad,lead", [(1000, 3, 0), (1000, 0, 1), (33, 7, 5), (128256, 1, 3)])
def test_strides_and_starts_bf16(lib, V, pad, lead):
    import torch
    g = np.random.default_rng(V + pad)
    raw = torch.tensor(g.normal(0, 2, 5 * (V + pad) + lead), dtype=torch.bfloat16, device="cuda")
    x = raw[lead:].view(5, V + pad)[:, :V]
    us = [0.1, 0.3, 0.5, 0.7, 0.9]
    ids, lp = sample_gpu(lib, x, "bf16", 0.9, 50, 0.9, 0.01, us)
    same, lps = sample_gpu(lib, x.contiguous(), "bf16", 0.9, 50, 0.9, 0.01, us)
    assert ids.tolist() == same.tolist() and lp.tolist() == lps.tolist()
    for r, u in enumerate(us):
        want = sample_plain(x[r].double().cpu().numpy(), float(np.float32(0.9)), 50, float(np.float32(0.9)),
                            float(np.float32(0.01)), float(np.float32(u)))
        assert want[2] < V * 2.0 ** -44 or ids[r] == want[0]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_16_bit_row_does_not_depend_on_its_batch(lib, dtype):
    import torch
    g = np.random.default_rng(11)
    x = torch.tensor(g.normal(0, 2, (300, 40000)), dtype=torch_type(dtype), device="cuda")
    T, k, p, mp = g.choice([0.7, 1.0, 1.4], 300), g.choice([0, 50, 1500], 300), g.choice([1.0, 0.9], 300), g.choice([0.0, 0.02], 300)
    u = g.random(300)
    ids, lp = sample_gpu(lib, x, dtype, T, k, p, mp, u)
    for lo, hi in ((0, 1), (7, 8), (100, 108), (40, 120)):
        i, l = sample_gpu(lib, x[lo:hi], dtype, T[lo:hi], k[lo:hi], p[lo:hi], mp[lo:hi], u[lo:hi],
                          stream=torch.cuda.Stream())
        assert (i == ids[lo:hi]).all() and (l.view(np.uint32) == lp[lo:hi].view(np.uint32)).all()
