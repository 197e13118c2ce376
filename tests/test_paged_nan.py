"""llmq_paged_attention with NaN and infinities in what it uses: the heads they reach say so
in the output and in lse, which a row without positions does not share; all others are as
they were."""
from __future__ import annotations

import numpy as np
import pytest

from paged_helpers import attend_gpu, make_pool, torch_type

gpu = pytest.mark.gpu
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


def state(dtype, kv_dtype, lens, H, KV, hd, page):
    import torch
    g = torch.Generator().manual_seed(3)
    need = [-(-n // page) for n in lens]
    k, v = make_pool(sum(need) + 1, page, KV, hd, kv_dtype, seed=5)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randn((len(lens), H, hd), generator=g).to(torch_type(dtype)).cuda()
    return k, v, q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("lens", [[5, 0, 40, 17], [3000, 0, 700, 2999]], ids=["short", "split"])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (6, 2, 48), (20, 2, 128)])
@pytest.mark.parametrize("what", ["q", "key", "value"])
def test_nan_reaches_its_heads_alone(lib, dtype, kv_dtype, lens, H, KV, hd, what):
    import torch
    k, v, q, table, n = state(dtype, kv_dtype, lens, H, KV, hd, 16)
    out0, lse0, _ = attend_gpu(lib, k, v, kv_dtype, q, table, n, dtype)
    bad = torch.zeros((len(lens), H), dtype=torch.bool)
    r, pos, G = 2, lens[2] - 3, H // KV
    if what == "q":
        q[r, 3, 5] = float("nan")
        bad[r, 3] = True
    else:
        (k if what == "key" else v)[int(table[r, pos // 16]), pos % 16, 1, 5] = float("nan")
        bad[r, G:2 * G] = True
    out, lse, status = attend_gpu(lib, k, v, kv_dtype, q, table, n, dtype)
    bad, good = bad.cuda(), ~bad.cuda()
    assert status == 0
    assert torch.equal(out[good], out0[good]) and torch.equal(lse[good], lse0[good])
    assert torch.isneginf(lse[1]).all() and (out[1] == 0).all()
    if what == "value":  # a weight's product: its dim alone
        assert torch.isnan(out[bad][:, 5]).all() and torch.equal(lse[bad], lse0[bad])
    else:
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES[:3])
@pytest.mark.parametrize("lens", [[40], [3000]], ids=["short", "split"])
def test_infinite_keys(lib, dtype, kv_dtype, lens):
    """A +infinite score has no softmax: NaN.  A -infinite one leaves its position out."""
    import torch
    k, v, q, table, n = state(dtype, kv_dtype, lens, 4, 1, 64, 16)
    pos = lens[0] - 7
    page, tok = int(table[0, pos // 16]), pos % 16
    q[0, :, 9] = torch.tensor([1.0, -1.0, 2.0, -0.5])
    k[page, tok, 0] = 0.0
    k[page, tok, 0, 9] = float("inf")
    out, lse, _ = attend_gpu(lib, k, v, kv_dtype, q, table, n, dtype)
    assert torch.isnan(out[0, 0::2]).all() and torch.isnan(lse[0, 0::2]).all()
    seen = torch.tensor([p for p in range(lens[0]) if p != pos])
    pid = table[0].cpu()[seen // 16].long()
    K, V = k[pid, seen % 16, 0].double().cpu().numpy(), v[pid, seen % 16, 0].double().cpu().numpy()
    for h in (1, 3):
        s = K @ q[0, h].double().cpu().numpy() / 8.0
        w = np.exp(s - s.max())
        want = (w[:, None] * V).sum(0) / w.sum()
        half = torch.finfo(torch_type(dtype)).eps / 2
        # sums of n f32 terms, weights of 16 bits at least, whose exponents are good to 2^-17
        tol = (lens[0] * 2.0 ** -23 + 2.0 ** -15) * np.abs(V).max() + half * np.abs(want)
        assert (np.abs(out[0, h].double().cpu().numpy() - want) <= tol).all()
        assert abs(float(lse[0, h]) - (s.max() + np.log(w.sum()))) <= lens[0] * 2.0 ** -23 + 2.0 ** -19


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES[:3])
def test_all_scores_minus_infinite(lib, dtype, kv_dtype):
    """Nothing is left: as a row without positions.  (Over a 16-bit pool an f32 q is a sum of
    terms, some of them zero: its product with an infinity is NaN.)"""
    import torch
    k, v, q, table, n = state(dtype, kv_dtype, [37], 4, 1, 64, 16)
    q[0, :, 9] = -1.0
    k[:, :, 0] = 0.0
    k[:, :, 0, 9] = float("inf")
    out, lse, _ = attend_gpu(lib, k, v, kv_dtype, q, table, n, dtype)
    assert (out == 0).all() and torch.isneginf(lse).all()
