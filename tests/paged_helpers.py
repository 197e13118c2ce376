"""Plain 64-bit forms of the serving operators and small callers of the
library's, shared by their tests."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

import llmq

CODES = {"f32": llmq.LLMQ_F32, "f16": llmq.LLMQ_F16, "bf16": llmq.LLMQ_BF16}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def ok(lib, rc):
    assert rc == 0, lib.q_llama_last_error_message()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_of(stream):
    return None if stream is None else stream.cuda_stream


# --------------------------------------------------------------------- plan
def plan_plain(cached, added, page, max_pages, max_rows, free, head, table):
    """The documented rules, request by request."""
    n = len(cached)
    cap = page * max_pages
    lens, first, flags = [], [0], 0
    table = table.copy()
    rows_seen = pages_seen = taken = 0
    slots, pos, seqs = [], [], []
    plan = []
    bad_head = head < 0
    if bad_head:
        flags |= llmq.LLMQ_PAGED_NO_PAGES
    h0 = max(head, 0)
    for b in range(n):
        c, a = int(cached[b]), int(added[b])
        held = 0 <= c <= cap
        valid = held and a >= 0 and c + a <= cap
        if not valid:
            flags |= llmq.LLMQ_PAGED_BAD_LEN
        rows_seen += a if valid else 0
        fits = valid and (a == 0 or rows_seen <= max_rows)
        if valid and not fits:
            flags |= llmq.LLMQ_PAGED_NO_ROWS
        have = -(-c // page)
        need = -(-(c + a) // page) - have if fits else 0
        pages_seen += need
        served = fits and (need == 0 or (not bad_head and h0 + pages_seen <= len(free)))
        if fits and not served:
            flags |= llmq.LLMQ_PAGED_NO_PAGES
        if served:
            for i in range(need):
                table[b, have + i] = free[h0 + taken + i]
            taken += need
        mine = a if served else 0
        lens.append(c + mine if held else 0)
        first.append(first[-1] + mine)
        plan.append((b, c, mine))
    for b, c, mine in plan:
        for p in range(c, c + mine):
            pid = int(table[b, p // page])
            if pid < 0:
                flags |= llmq.LLMQ_PAGED_BAD_PAGE
            slots.append(pid * page + p % page if pid >= 0 else -1)
            pos.append(p)
            seqs.append(b)
    pad = max_rows - len(slots)
    return dict(table=table, lens=lens, first=first, slots=slots + [-1] * pad, positions=pos + [-1] * pad,
                seqs=seqs + [-1] * pad, spans=[p + 1 for p in pos] + [0] * pad,
                next_head=head if bad_head else h0 + taken, status=flags)


def plan_gpu(lib, cached, added, page, max_pages, max_rows, free, head, table, stream=None, alias=False):
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    n = len(cached)
    t = dict(cached=torch.tensor(cached, **i32), added=torch.tensor(added, **i32),
             free=torch.tensor(list(free), **i32), head=torch.tensor([head], **i32),
             table=torch.tensor(table, **i32), lens=torch.full((n,), -9, **i32), first=torch.full((n + 1,), -9, **i32),
             slots=torch.full((max_rows,), -9, dtype=torch.int64, device="cuda"),
             positions=torch.full((max_rows,), -9, **i32), seqs=torch.full((max_rows,), -9, **i32),
             spans=torch.full((max_rows,), -9, **i32), next_head=torch.full((1,), -9, **i32),
             status=torch.zeros(1, **i32))
    if alias:
        t["lens"], t["next_head"] = t["cached"], t["head"]
    a = llmq.PagedPlan(n_seqs=n, page_size=page, max_pages=max_pages, max_rows=max_rows, n_free=len(free),
                       cached=ptr(t["cached"]), added=ptr(t["added"]), free_pages=ptr(t["free"]),
                       free_head=ptr(t["head"]), table=ptr(t["table"]), table_stride=t["table"].stride(0) if n else max_pages,
                       lens=ptr(t["lens"]), first=ptr(t["first"]), slots=ptr(t["slots"]), positions=ptr(t["positions"]),
                       seqs=ptr(t["seqs"]), spans=ptr(t["spans"]), next_head=ptr(t["next_head"]),
                       status=ptr(t["status"]))
    torch.cuda.synchronize()
    ok(lib, lib.llmq_paged_plan(C.byref(a), stream_of(stream)))
    torch.cuda.synchronize()
    out = {k: t[k].cpu().numpy() for k in ("table", "lens", "first", "slots", "positions", "seqs", "spans")}
    out["next_head"], out["status"] = int(t["next_head"]), int(t["status"])
    return out


# --------------------------------------------------------------------- pool
def make_pool(pages, page, n_kv, hd, kv_dtype, order="token", seed=0, fill=None):
    """(k, v) as [page][token][head][d] views of pools laid out in `order`."""
    import torch
    g = torch.Generator().manual_seed(seed)
    shape = (pages, page, n_kv, hd) if order == "token" else (pages, n_kv, page, hd)
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g).to(torch_type(kv_dtype)) if fill is None else \
            torch.full(shape, fill, dtype=torch_type(kv_dtype))
        x = x.cuda()
        out.append(x if order == "token" else x.transpose(1, 2))
    return out


def describe_pool(k, v, kv_dtype):
    assert k.stride() == v.stride() and k.stride(3) == 1
    return llmq.PagedKV(k=ptr(k), v=ptr(v), dtype=CODES[kv_dtype], n_pages=k.shape[0], page_size=k.shape[1],
                        n_kv=k.shape[2], head_dim=k.shape[3], page_stride=k.stride(0), token_stride=k.stride(1),
                        head_stride=k.stride(2))


# ---------------------------------------------------------------- attention
def attend_descriptor(lib, k, q, out, table, lens, dtype, lse=None, seqs=None, window=0, scale=0.0, status=None):
    """(descriptor, workspace)"""
    import torch
    R, H, hd = q.shape
    need = lib.llmq_paged_attention_workspace(R, H, k.shape[2], hd)
    work = torch.full((max(need, 16),), 0x7f, dtype=torch.uint8, device="cuda")
    a = llmq.PagedAttention(n_rows=R, n_heads=H, dtype=CODES[dtype], window=window, max_pages=table.shape[1],
                            n_seqs=table.shape[0], scale=scale, q=ptr(q), q_stride=q.stride(0), out=ptr(out),
                            out_stride=out.stride(0), lse=ptr(lse), table=ptr(table), table_stride=table.stride(0),
                            seqs=ptr(seqs), lens=ptr(lens), workspace=ptr(work), workspace_bytes=need,
                            status=ptr(status))
    return a, work


def attend_gpu(lib, k, v, kv_dtype, q, table, lens, dtype, stream=None, **kw):
    """(out, lse, status)"""
    import torch
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv = describe_pool(k, v, kv_dtype)
    a, work = attend_descriptor(lib, k, q, out, table, lens, dtype, lse=lse, status=status, **kw)
    torch.cuda.synchronize()
    ok(lib, lib.llmq_paged_attention(C.byref(kv), C.byref(a), stream_of(stream)))
    torch.cuda.synchronize()
    return out, lse, int(status)


def attend_plain(k, v, q, table, lens, seqs=None, window=0, scale=0.0):
    """(out, lse, their bounds, max|v|): 64 bits on the CPU, and how far an f32
    evaluation may be from it before the output is rounded.

    A score is a sum of hd products and one scaling: off by at most (hd + 3)
    2^-24 scale sum|q||k|.  Its exponential, as 2^(s log2 e): the product with
    log2 e moves the exponent by 2^-23 |s - m| + 2^-23 |s|, the device's ex2 is
    good to 2^-22; so a weight's relative error is at most
    e = ds + 2^-22 (1 + |s|max + |s - m|max), the same again through the maximum's own
    error.  Sums of n weights and of n weighted values in any order are off by n 2^-24
    of the sum of magnitudes, and joining partial results over at most 64 more
    factors by 64 2^-23.  The quotient: |do| <= (2 (2 e + n 2^-24 + 64 2^-23) + 2^-23) max|v|,
    and lse by the sum's relative error and a rounding of its own size."""
    kc, vc, qc = k.double().cpu(), v.double().cpu(), q.double().cpu()
    tb, ln = table.cpu().numpy(), lens.cpu().numpy()
    R, H, hd = qc.shape
    P, page, n_kv = kc.shape[:3]
    G = H // n_kv
    scale = scale or 1.0 / math.sqrt(hd)
    out, lse = np.zeros((R, H, hd)), np.full((R, H), -np.inf)
    bo, bl, vm = np.zeros((R, H, 1)), np.zeros((R, H)), np.zeros((R, H, 1))
    for r in range(R):
        s = r if seqs is None else int(seqs[r])
        n = int(ln[r])
        if s < 0 or s >= tb.shape[0] or n <= 0:
            continue
        n = min(n, tb.shape[1] * page)
        p = np.arange(max(0, n - window) if window else 0, n)
        pid = tb[s, p // page]
        good = (pid >= 0) & (pid < P)
        p, pid = p[good], pid[good]
        if not len(p):
            continue
        K, V = kc[pid, p % page].numpy(), vc[pid, p % page].numpy()  # [n, n_kv, hd]
        for h in range(H):
            x = qc[r, h].numpy()
            prods = K[:, h // G] * x
            sc = prods.sum(1) * scale
            m = sc.max()
            e = np.exp(sc - m)
            out[r, h] = (e[:, None] * V[:, h // G]).sum(0) / e.sum()
            lse[r, h] = m + np.log(e.sum())
            ds = (hd + 3) * 2.0 ** -24 * scale * np.abs(prods).sum(1).max()
            er = ds + 2.0 ** -22 * (1 + np.abs(sc).max() + (m - sc).max())
            rel = 2 * er + len(p) * 2.0 ** -24 + 64 * 2.0 ** -23
            vm[r, h] = np.abs(V[:, h // G]).max()
            bo[r, h] = (2 * rel + 2.0 ** -23) * vm[r, h]
            bl[r, h] = rel + 2.0 ** -22 * (1 + abs(lse[r, h]))
    return out, lse, bo, bl, vm


def check_attend(out, lse, plain, dtype, kv_dtype):
    """The output's rounding adds half a step of its type.  Over a 16-bit pool a weight
    is a sum of 16-bit terms, off by half a step of the last one: 2^-16 (two bf16
    terms), 2^-24 (three) or 2^-22 (two of f16) of itself, so the output by that times
    max|v|."""
    import torch
    o, l, bo, bl, vm = plain
    half = torch.finfo(torch_type(dtype)).eps / 2
    terms = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -24 if dtype == "f32" else 2.0 ** -16}[kv_dtype]
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    tol = bo + terms * vm
    tol = tol + half * (np.abs(o) + tol) + (2.0 ** -25 if dtype == "f16" else 1e-30)  # the least f16 step is 2^-24
    assert np.isfinite(got).all()
    off = np.abs(got - o)
    assert (off <= tol).all(), f"{(off > tol).sum()} outputs off, worst {(off / tol).max()} of the bound"
    empty = np.isneginf(l)
    assert np.isneginf(gl[empty]).all() and (got[empty] == 0).all()
    assert (np.abs(gl[~empty] - l[~empty]) <= bl[~empty]).all()


# ----------------------------------------------------------------- sampling
def sample_plain(row, T, top_k, top_p, min_p, u):
    """(id, log share, margin): the documented rules in 64 bits.  margin is how far u is
    from where the drawn token changes, and each cut from where what it keeps
    changes, as a share of the whole sum."""
    row = np.asarray(row, np.float64)
    usable = ~np.isnan(row) & ~np.isneginf(row)
    if not usable.any():
        return -1, -np.inf, np.inf
    mx = row[usable].max()
    if not T > 0:
        return int(np.flatnonzero(usable & (row == mx))[0]), 0.0, np.inf
    idx = np.flatnonzero(usable)
    order = idx[np.argsort(-row[idx], kind="stable")]
    x = row[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == mx, 1.0, 0.0 if np.isposinf(mx) else np.exp((x - mx) / np.float64(T)))
    S = np.cumsum(w.astype(np.longdouble))
    n, margin = len(order), np.inf
    total = S[-1]
    if 0 < top_k < n:
        n = top_k
    if min_p > 0:
        mp = min(float(min_p), 1.0)
        n = min(n, int((w >= mp).sum()))
        if mp < 1.0:
            margin = min(margin, float(np.abs(w[w < 1.0] - mp).min()) if (w < 1.0).any() else np.inf)
    if 0 < top_p < 1:
        t = np.longdouble(np.float32(top_p)) * total
        n = min(n, int(np.searchsorted(S, t)) + 1)
        margin = min(margin, float(np.abs(S - t).min() / total))
    n = max(n, 1)
    uu = 0.0 if not u > 0 else min(float(u), 1.0)
    t = np.longdouble(uu) * S[n - 1]
    at = min(int(np.searchsorted(S, t)), n - 1)
    near = S[:n] if uu < 1 else S[:n - 1]  # at u = 1 the sum itself is reached, whatever it is
    if uu > 0 and len(near):
        margin = min(margin, float(np.abs(near - t).min() / total))
    return int(order[at]), float(np.log(w[at] / S[n - 1])), margin


def sample_gpu(lib, logits, dtype, T=None, top_k=None, top_p=None, min_p=None, u=None, stream=None, want=True):
    import torch
    f = dict(dtype=torch.float32, device="cuda")
    R, V = logits.shape

    def col(x, **kw):
        return None if x is None else torch.tensor(np.broadcast_to(np.asarray(x), (R,)).copy(), **kw)

    t = [col(T, **f), col(top_k, dtype=torch.int32, device="cuda"), col(top_p, **f), col(min_p, **f), col(u, **f)]
    ids = torch.full((R,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((R,), 7.0, **f) if want else None
    a = llmq.SampleRows(n_rows=R, vocab=V, dtype=CODES[dtype], logits=ptr(logits), stride=logits.stride(0),
                        temperature=ptr(t[0]), top_k=ptr(t[1]), top_p=ptr(t[2]), min_p=ptr(t[3]), u=ptr(t[4]),
                        ids=ptr(ids), logprobs=ptr(lp))
    torch.cuda.synchronize()
    ok(lib, lib.llmq_sample_rows(C.byref(a), stream_of(stream)))
    torch.cuda.synchronize()
    return ids.cpu().numpy(), None if lp is None else lp.cpu().numpy()
