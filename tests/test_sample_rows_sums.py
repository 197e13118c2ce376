"""llmq_sample_rows where its sums have to agree to the unit: the last token of what is
kept, reached by u = 1, in rows whose weights are formed at several places (a histogram of
a cluster's slices, a list, divided steps, counts of values)."""
from __future__ import annotations

import numpy as np
import pytest

from paged_helpers import sample_gpu, torch_type

gpu = pytest.mark.gpu


def rows_of(V, seed):
    """Few distinct values, all distinct ones, and a few high ones above a body of ties."""
    g = np.random.default_rng(seed)
    few = g.choice([0.0, -0.37, -1.1], V)
    some = np.round(g.normal(0, 1, V), 1)
    smooth = g.normal(0, 1, V)
    body = np.full(V, -2.3)
    body[g.integers(0, V, 50)] = g.uniform(-1, 0, 50)
    heavy_last = np.where(np.arange(V) < V // 3, 0.011, -0.017)
    return [few, some, smooth, body, heavy_last]


def last_of(row, T, k):
    """(id, log share) of the last token kept: the kth, or the last of all, in falling order."""
    order = np.argsort(-row, kind="stable")
    n = k if 0 < k < len(row) else len(row)
    w = np.exp((row[order] - row[order[0]]) / T)
    return int(order[n - 1]), float(np.log(w[n - 1] / w[:n].sum()))


def check_last(lib, rows, dtype, temps, ks):
    import torch
    t = torch.tensor(np.stack(rows).astype(np.float32)).to(torch_type(dtype))
    seen, x = t.double().numpy(), t.cuda()
    V = seen.shape[1]
    for T in temps:
        Tf = float(np.float32(T))
        if ((seen.max(1) - seen.min(1)) / Tf).max() > 20:
            continue  # every weight is far above what rounds to nothing: the last token has one
        for k in ks:
            ids, lp = sample_gpu(lib, x, dtype, T, k, 1.0, 0.0, 1.0)
            for r in range(len(rows)):
                i, l = last_of(seen[r], Tf, k)
                assert ids[r] == i, (r, T, k)
                # the kept sum, at least 1, is off by half of 2^-42 a token at most; the log is rounded to f32
                assert abs(lp[r] - l) <= 2.0 ** -23 * (1 + abs(l)) + V * 2.0 ** -43, (r, T, k)
            one, _ = sample_gpu(lib, x.repeat(60, 1), dtype, T, k, 1.0, 0.0, 1.0)  # a CTA a row, all at once
            assert (one.reshape(60, -1) == ids).all(), (T, k)


TEMPS = [0.3, 0.5, 0.61, 0.77, 1.0, 1.0001, 1.37, 2.0, 2.9, 5.3, 11.0, 33.0, 100.0, 1234.5, 1e5, 1e9]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [70, 2048, 2049, 5000, 32000, 50257])
def test_the_last_token_without_cuts(lib, V, dtype):
    check_last(lib, rows_of(V, V), dtype, TEMPS, [0])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_the_last_token_of_a_top_k(lib, dtype):
    V = 9001
    check_last(lib, rows_of(V, 4), dtype, TEMPS[::3], [1, 40, 97, 2048, 3001, 9000])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_the_last_token_of_ties(lib, dtype):
    """Rows of one value and of two: steps that no list holds."""
    V = 40000
    two = np.where(np.random.default_rng(2).random(V) < 0.5, 1.0, 0.25)
    check_last(lib, [np.full(V, 0.5), two, two[::-1].copy()], dtype, TEMPS, [0, 2049, 30001])
