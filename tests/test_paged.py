"""The paged key-value cache: llmq_paged_plan, llmq_paged_append and
llmq_paged_attention against plain 64-bit forms, at the sizes and masks where
they can go wrong, and their refusals (which need no GPU)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import llmq
from conftest import has_gpu
from paged_helpers import (CODES, attend_descriptor, attend_gpu, attend_plain, check_attend, describe_pool, make_pool,
                           ok, plan_gpu, plan_plain, ptr, torch_type)

gpu = pytest.mark.gpu
F = 0x10000  # a pointer that no check before the GPU's looks behind


# ----------------------------------------------------------- refusals (CPU)
def pool_args(**kw):
    d = dict(k=F, v=F, dtype=0, n_pages=4, page_size=16, n_kv=2, head_dim=64, page_stride=2048, token_stride=128,
             head_stride=64)
    d.update(kw)
    return llmq.PagedKV(**d)


def plan_args(**kw):
    d = dict(n_seqs=2, page_size=16, max_pages=4, max_rows=8, n_free=3, cached=F, added=F, free_pages=F, table=F,
             table_stride=4, lens=F, first=F, slots=F)
    d.update(kw)
    return llmq.PagedPlan(**d)


def append_args(**kw):
    d = dict(n_rows=3, n_heads=4, dtype=0, rope_len=32, q=F, k=F, v=F, q_stride=256, k_stride=128, v_stride=128,
             q_out=F, q_out_stride=256, slots=F, positions=F, rope_cos=F, rope_sin=F)
    d.update(kw)
    return llmq.PagedAppend(**d)


def attend_args(**kw):
    d = dict(n_rows=3, n_heads=4, dtype=0, max_pages=4, n_seqs=3, q=F, q_stride=256, out=F, out_stride=256, table=F,
             table_stride=4, lens=F, workspace=F, workspace_bytes=1 << 40)
    d.update(kw)
    return llmq.PagedAttention(**d)


def refused(lib, fn, *args):
    lib.q_llama_clear_error()
    rc = fn(*[C.byref(a) if a is not None else None for a in args], None)
    assert rc == llmq.LLMQ_ERR_ARG == lib.q_llama_last_error()
    assert lib.q_llama_last_error_message().startswith(fn.__name__.encode())
    lib.q_llama_clear_error()


BAD_POOLS = [dict(k=None), dict(v=None), dict(dtype=3), dict(dtype=-1), dict(n_pages=0), dict(page_size=0),
             dict(n_pages=1 << 20, page_size=1 << 11), dict(n_kv=0), dict(head_dim=0), dict(head_dim=60),
             dict(head_dim=264), dict(k=F + 8), dict(v=F + 4), dict(page_stride=2046), dict(token_stride=-128),
             dict(head_stride=66)]


@pytest.mark.parametrize("bad", [dict(n_seqs=-1), dict(max_rows=-1), dict(n_free=-1), dict(page_size=0),
                                 dict(max_pages=0), dict(page_size=1 << 16, max_pages=1 << 16, table_stride=1 << 16),
                                 dict(table_stride=3), dict(cached=None), dict(added=None), dict(table=None),
                                 dict(lens=None), dict(first=None), dict(slots=None), dict(free_pages=None)], ids=str)
def test_plan_refuses(lib, bad):
    refused(lib, lib.llmq_paged_plan, plan_args(**bad))


@pytest.mark.parametrize("bad", [dict(n_rows=-1), dict(n_heads=-1), dict(dtype=7), dict(k=None), dict(v=None),
                                 dict(slots=None), dict(q=None), dict(q_out=None), dict(n_heads=0), dict(rope_sin=None),
                                 dict(positions=None), dict(rope_len=0), dict(k_stride=127), dict(v_stride=64),
                                 dict(q_stride=255), dict(q_out_stride=1), dict(k=F + 2), dict(dtype=1)], ids=str)
def test_append_refuses(lib, bad):
    refused(lib, lib.llmq_paged_append, pool_args(), append_args(**bad))


@pytest.mark.parametrize("bad", [dict(n_rows=-1), dict(n_heads=0), dict(n_heads=3), dict(dtype=2), dict(window=-1),
                                 dict(max_pages=-1), dict(max_pages=1 << 28, table_stride=1 << 28), dict(table_stride=3),
                                 dict(scale=float("inf")), dict(scale=float("nan")), dict(q=None), dict(out=None),
                                 dict(lens=None), dict(table=None), dict(n_seqs=2), dict(q_stride=255),
                                 dict(out_stride=8), dict(q=F + 1), dict(workspace=None), dict(workspace=F + 8),
                                 dict(workspace_bytes=0)], ids=str)
def test_attention_refuses(lib, bad):
    refused(lib, lib.llmq_paged_attention, pool_args(), attend_args(**bad))


@pytest.mark.parametrize("bad", BAD_POOLS, ids=str)
def test_pool_refused(lib, bad):
    refused(lib, lib.llmq_paged_append, pool_args(**bad), append_args())
    refused(lib, lib.llmq_paged_attention, pool_args(**bad), attend_args())


def test_null_descriptors_and_workspace_sizes(lib):
    refused(lib, lib.llmq_paged_plan, None)
    refused(lib, lib.llmq_paged_append, None, append_args())
    refused(lib, lib.llmq_paged_append, pool_args(), None)
    refused(lib, lib.llmq_paged_attention, pool_args(), None)
    for sizes in [(-1, 4, 2, 64), (1, 0, 1, 64), (1, 4, 3, 64), (1, 4, 2, 0), (1, 4, 2, 260), (1, 4, 2, 257)]:
        assert lib.llmq_paged_attention_workspace(*sizes) == 0
        assert lib.q_llama_last_error() == llmq.LLMQ_ERR_ARG
        lib.q_llama_clear_error()
    assert lib.llmq_paged_attention_workspace(64, 32, 8, 128) > 0


def test_empty_calls_need_no_gpu(lib):
    assert lib.llmq_paged_append(C.byref(pool_args()), C.byref(append_args(n_rows=0)), None) == 0
    assert lib.llmq_paged_attention(C.byref(pool_args()), C.byref(attend_args(n_rows=0)), None) == 0


@pytest.mark.skipif(has_gpu(), reason="this machine has a GPU")
def test_good_calls_without_a_gpu_say_so(lib):
    for rc in (lib.llmq_paged_plan(C.byref(plan_args()), None),
               lib.llmq_paged_append(C.byref(pool_args()), C.byref(append_args()), None),
               lib.llmq_paged_attention(C.byref(pool_args()), C.byref(attend_args()), None)):
        assert rc == llmq.LLMQ_ERR_NO_DEVICE
    lib.q_llama_clear_error()


def test_plain_plan_on_a_case_by_hand():
    t = np.array([[5, -1, -1], [-1, -1, -1]])
    p = plan_plain([3, 0], [2, 3], 4, 3, 6, [8, 9, 7], 1, t)
    assert p["table"].tolist() == [[5, 9, -1], [7, -1, -1]]
    assert p["slots"] == [23, 36, 28, 29, 30, -1] and p["positions"] == [3, 4, 0, 1, 2, -1]
    assert p["first"] == [0, 2, 5] and p["lens"] == [5, 3] and p["next_head"] == 3 and p["status"] == 0


# -------------------------------------------------------------------- plan
def check_plan(lib, *args, **kw):
    got, want = plan_gpu(lib, *args, **kw), plan_plain(*args)
    for k in ("table", "lens", "first", "slots", "positions", "seqs", "spans"):
        np.testing.assert_array_equal(got[k].reshape(-1), np.asarray(want[k]).reshape(-1), err_msg=k)
    assert got["next_head"] == want["next_head"] and got["status"] == want["status"]
    return want


def random_plan(seed, n, page, max_pages, big):
    rng = np.random.default_rng(seed)
    cap = page * max_pages
    cached = rng.integers(0, cap + 1, n)
    added = np.minimum(rng.integers(0, 1 + big, n), cap - cached)
    table = np.full((n, max_pages), -1)
    have = -(-cached // page)
    pages = rng.permutation(int(have.sum()) + int((-(-(cached + added) // page) - have).sum()) + 3)
    at = 0
    for b in range(n):
        table[b, :have[b]] = pages[at:at + have[b]]
        at += have[b]
    return cached.tolist(), added.tolist(), pages[at:].tolist(), table


@gpu
@pytest.mark.parametrize("n,page,max_pages,big", [(1, 16, 4, 1), (3, 1, 5, 3), (64, 16, 136, 1), (31, 24, 9, 70),
                                                  (1023, 8, 6, 4), (1024, 8, 6, 4), (1025, 7, 6, 40), (3001, 16, 3, 5)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(lib, n, page, max_pages, big, alias):
    cached, added, free, table = random_plan(n * 7 + page, n, page, max_pages, big)
    want = check_plan(lib, cached, added, page, max_pages, sum(added) + 5, free, 0, table, alias=alias)
    assert want["status"] == 0


@gpu
def test_plan_many_rows_of_one_request(lib):
    check_plan(lib, [5, 0, 7], [1, 40000, 1], 16, 2600, 40007, list(range(3000)), 2, np.arange(3 * 2600).reshape(3, -1))


@gpu
@pytest.mark.parametrize("n", [4, 1500])
def test_plan_runs_out(lib, n):
    cached, added, free, table = random_plan(n, n, 8, 6, 20)
    rows = sum(added)
    for max_rows, keep, head in [(rows // 2, len(free), 0), (rows, len(free) // 2, 0), (rows // 3, len(free) // 4, 1),
                                 (0, len(free), 0), (rows, 0, 0), (rows, len(free), len(free)), (rows, len(free), -2),
                                 (rows, len(free), len(free) + 9)]:
        check_plan(lib, cached, added, 8, 6, max_rows, free[:keep], head, table)


@gpu
def test_plan_bad_lengths_and_missing_pages(lib):
    cached = [-1, 3, 49, 48, 10, 47, 2**31 - 1, 20]
    added = [1, -2, 0, 1, 39, 1, 2**31 - 1, 3]
    table = np.full((8, 6), -1)
    table[4, :2] = [3, 4]
    table[5] = [5, 6, 7, 8, 9, 10]
    want = check_plan(lib, cached, added, 8, 6, 64, [20, 21, 22, 23], 0, table)
    assert want["lens"] == [0, 3, 0, 48, 10, 48, 0, 23] or want["lens"][5] == 48
    assert want["status"] & llmq.LLMQ_PAGED_BAD_LEN and want["status"] & llmq.LLMQ_PAGED_BAD_PAGE


@gpu
def test_plan_without_requests_or_optional_outputs(lib):
    import torch
    check_plan(lib, [], [], 8, 6, 5, [1, 2], 1, np.zeros((0, 6)))
    i32 = dict(dtype=torch.int32, device="cuda")
    z = torch.tensor([7], **i32)
    table, lens, first = torch.zeros((1, 2), **i32), torch.zeros(1, **i32), torch.zeros(2, **i32)
    slots, free = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.tensor([5], **i32)
    a = llmq.PagedPlan(n_seqs=1, page_size=8, max_pages=2, max_rows=3, n_free=1, cached=ptr(z), added=ptr(z * 0 + 2),
                       free_pages=ptr(free), table=ptr(table), table_stride=2, lens=ptr(lens), first=ptr(first),
                       slots=ptr(slots))
    added = torch.tensor([2], **i32)
    a.added = ptr(added)
    ok(lib, lib.llmq_paged_plan(C.byref(a), None))
    torch.cuda.synchronize()
    assert slots.tolist() == [7, 40, -1] and first.tolist() == [0, 2] and table.tolist() == [[0, 5]]


# ------------------------------------------------------------------ append
def append_plain(s, turn=True):
    """(k, v, q) in 64 bits, unrounded; untouched elements as they were."""
    x, KV, H, hd = s["qkv"].double().cpu(), s["n_kv"], s["heads"], s["hd"]
    T, half = x.shape[0], hd // 2
    x = x.view(T, -1, hd)
    k, v, q = s["k"].double().cpu().clone(), s["v"].double().cpu().clone(), s["q_out"].double().cpu().clone()
    cos, sin = s["cos"].double().cpu(), s["sin"].double().cpu()
    page = k.shape[1]
    for t in range(T):
        slot = int(s["slots"][t])
        if slot < 0 or slot >= k.shape[0] * page:
            continue
        y = x[t].clone()
        if turn:
            p = int(s["positions"][t])
            if p < 0 or p >= cos.shape[0]:
                continue
            a, b = x[t, :H + KV, :half], x[t, :H + KV, half:]
            y[:H + KV, :half] = a * cos[p] - b * sin[p]
            y[:H + KV, half:] = b * cos[p] + a * sin[p]
        q[t], k[slot // page, slot % page], v[slot // page, slot % page] = y[:H], y[H:H + KV], y[H + KV:]
    return k, v, q


def append_state(T, H, KV, hd, page, dtype, kv_dtype, order="token", seed=1, pad=0, lead=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    pages = T // page + 3
    width = (H + 2 * KV) * hd + pad
    raw = torch.randn(T * width + lead, generator=g).to(torch_type(dtype)).cuda()
    qkv = raw[lead:].view(T, width)[:, :(H + 2 * KV) * hd]
    k, v = make_pool(pages, page, KV, hd, kv_dtype, order, seed + 1)
    ang = torch.rand((50, hd // 2), generator=g) * 6
    return dict(qkv=qkv, k=k, v=v, n_kv=KV, heads=H, hd=hd, kv_dtype=kv_dtype, dtype=dtype,
                slots=torch.randperm(pages * page, generator=g)[:T].cuda(),
                positions=torch.randint(0, 50, (T,), generator=g, dtype=torch.int32).cuda(),
                cos=torch.cos(ang).cuda().contiguous(), sin=torch.sin(ang).cuda().contiguous(),
                q_out=torch.full((T, H, hd), 3.0).to(torch_type(dtype)).cuda(), raw=raw)


def append_call(lib, s, turn=True, with_q=True, status=None, stream=None, q_out=None):
    x, H, KV, hd, e = s["qkv"], s["heads"], s["n_kv"], s["hd"], s["qkv"].element_size()
    kv = describe_pool(s["k"], s["v"], s["kv_dtype"])
    qo = s["q_out"] if q_out is None else q_out
    a = llmq.PagedAppend(n_rows=x.shape[0], n_heads=H if with_q else 0, dtype=CODES[s["dtype"]],
                         rope_len=s["cos"].shape[0] if turn else 0, q=x.data_ptr() if with_q else None,
                         k=x.data_ptr() + H * hd * e, v=x.data_ptr() + (H + KV) * hd * e,
                         q_stride=x.stride(0) if with_q else 0, k_stride=x.stride(0), v_stride=x.stride(0),
                         q_out=qo.data_ptr() if with_q else None, q_out_stride=qo.stride(0) if with_q else 0,
                         slots=ptr(s["slots"]), positions=ptr(s["positions"]), rope_cos=ptr(s["cos"]) if turn else None,
                         rope_sin=ptr(s["sin"]) if turn else None, status=ptr(status))
    ok(lib, lib.llmq_paged_append(C.byref(kv), C.byref(a), None if stream is None else stream.cuda_stream))


def check_append(s, want):
    """Two products and a sum in f32, each off by half a step of at most
    |a| + |b| <= 2^3 here (normal numbers below 2^3, angles below 1): 3 * 2^3 *
    2^-24; then half a step of the stored type."""
    import torch
    for name, x in zip(("k", "v", "q_out"), want):
        got = s[name].double().cpu()
        half = torch.finfo(s[name].dtype).eps / 2
        tol = 24 * 2.0 ** -24 + half * (x.abs() + 24 * 2.0 ** -24)
        assert ((got - x).abs() <= tol).all(), name


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                                            ("f16", "f16")])
@pytest.mark.parametrize("T,H,KV,hd,page,order", [(1, 6, 2, 48, 16, "token"), (5, 1, 1, 8, 1, "head"),
                                                  (37, 8, 2, 128, 24, "head"), (130, 4, 4, 80, 7, "token"),
                                                  (9, 14, 2, 72, 16, "token"), (3, 3, 3, 256, 5, "head")])
def test_append(lib, T, H, KV, hd, page, order, dtype, kv_dtype):
    import torch
    s = append_state(T, H, KV, hd, page, dtype, kv_dtype, order)
    want = append_plain(s)
    append_call(lib, s)
    torch.cuda.synchronize()
    check_append(s, want)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,lead", [(1, 0), (8, 0), (0, 1), (3, 5)])
def test_append_odd_strides_and_starts(lib, dtype, pad, lead):
    import torch
    s = append_state(11, 4, 2, 64, 16, dtype, dtype, pad=pad, lead=lead)
    want = append_plain(s)
    append_call(lib, s)
    torch.cuda.synchronize()
    check_append(s, want)


@gpu
def test_append_padding_bad_slots_and_positions(lib):
    import torch
    s = append_state(40, 4, 2, 64, 16, "f32", "bf16")
    n = s["k"].shape[0] * 16
    s["slots"][[0, 7]] = -1
    s["slots"][3], s["slots"][4] = n, 2 ** 40
    s["positions"][9], s["positions"][10] = -1, 50
    want = append_plain(s)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    append_call(lib, s, status=status)
    torch.cuda.synchronize()
    check_append(s, want)
    assert int(status) == llmq.LLMQ_PAGED_BAD_SLOT | llmq.LLMQ_PAGED_BAD_POS
    assert (s["q_out"][[0, 3, 4, 7, 9, 10]] == 3.0).all()


@gpu
def test_append_without_angles_without_q_and_in_place(lib):
    import torch
    s = append_state(13, 4, 2, 64, 16, "f32", "f32")
    want = append_plain(s, turn=False)
    append_call(lib, s, turn=False)
    torch.cuda.synchronize()
    for n, w in zip(("k", "v", "q_out"), want):
        assert torch.equal(s[n].double().cpu(), w)  # copies
    s = append_state(13, 4, 2, 64, 16, "f32", "f32")
    want = append_plain(s)
    append_call(lib, s, with_q=False)
    torch.cuda.synchronize()
    assert (s["q_out"] == 3.0).all()
    s["q_out"].copy_(want[2])
    check_append(s, want)
    s = append_state(13, 4, 2, 64, 16, "f32", "f32")
    want = append_plain(s)
    append_call(lib, s, q_out=s["qkv"])  # q turned where it stands
    torch.cuda.synchronize()
    s["q_out"] = s["qkv"][:, :256].reshape(13, 4, 64)
    check_append(s, want)


# --------------------------------------------------------------- attention
def attend_state(lens, H, KV, hd, page, dtype, kv_dtype, order="token", seed=3, spare=2, width=None):
    import torch
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = perm[at:at + m]
        at += m
    k, v = make_pool(pages, page, KV, hd, kv_dtype, order, seed + 1)
    q = torch.randn((len(lens), H, hd), generator=g).to(torch_type(dtype)).cuda()
    return k, v, q, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]


def run_attend(lib, st, dtype, kv_dtype, **kw):
    k, v, q, table, lens = st
    out, lse, flags = attend_gpu(lib, k, v, kv_dtype, q, table, lens, dtype, **kw)
    kw.pop("stream", None)
    if kw.get("seqs") is not None:
        kw["seqs"] = kw["seqs"].cpu()
    check_attend(out, lse, attend_plain(k, v, q, table, lens, **kw), dtype, kv_dtype)
    return out, lse, flags


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,page,order", [(6, 2, 48, 16, "token"), (8, 1, 128, 24, "head"), (4, 4, 64, 1, "token"),
                                                (14, 2, 72, 7, "token"), (5, 1, 256, 32, "head"), (3, 3, 8, 64, "head"),
                                                (32, 2, 96, 16, "token"), (40, 1, 80, 16, "head"), (2, 1, 200, 5, "token")])
def test_attention(lib, H, KV, hd, page, order, dtype, kv_dtype):
    st = attend_state([1, 0, 17, 63, 64, 65, 130, 511], H, KV, hd, page, dtype, kv_dtype, order)
    assert run_attend(lib, st, dtype, kv_dtype)[2] == 0


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
def test_attention_every_short_length(lib, dtype, kv_dtype):
    run_attend(lib, attend_state(list(range(0, 140)), 4, 2, 64, 16, dtype, kv_dtype), dtype, kv_dtype)


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 5000), (3, 2049), (1, 20011)])
def test_attention_long(lib, rows, n, dtype, kv_dtype):
    run_attend(lib, attend_state([n] + [n // 3] * (rows - 1), 8, 2, 128, 16, dtype, kv_dtype), dtype, kv_dtype)


@gpu
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 1000])
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_window(lib, window, dtype, kv_dtype):
    run_attend(lib, attend_state([0, 1, 16, 17, 99, 100, 101, 700], 8, 2, 64, 24, dtype, kv_dtype), dtype, kv_dtype,
               window=window)


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
def test_attention_never_reads_past_a_row(lib, dtype, kv_dtype):
    """NaN and infinities past each length, in spare pages and in padded table entries."""
    import torch
    st = attend_state([1, 15, 16, 17, 40, 100], 8, 2, 64, 24, dtype, kv_dtype)
    k, v, q, table, lens = st
    want = attend_plain(k, v, q, table, lens)
    for x in (k, v):
        y = torch.full_like(x, float("nan"))
        y[:, ::2] = float("inf")
        for b, n in enumerate(lens.tolist()):
            for p in range(n):
                y[table[b, p // 24].long(), p % 24] = x[table[b, p // 24].long(), p % 24]
        x.copy_(y)
    table[table < 0] = 2 ** 30
    out, lse, flags = attend_gpu(lib, k, v, kv_dtype, q, table, lens, dtype)
    check_attend(out, lse, want, dtype, kv_dtype)
    assert flags == 0


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
def test_attention_bad_pages_lengths_and_rows(lib, dtype, kv_dtype):
    import torch
    st = attend_state([50, 60, 33, 70, 20, 64], 8, 2, 64, 16, dtype, kv_dtype, width=5)
    k, v, q, table, lens = st
    table[0, 1], table[1, 3], table[2, 0] = -1, k.shape[0], 2 ** 31 - 1
    table[2, 1], table[2, 2] = -5, -1  # a row of bad pages only
    lens[3], lens[4] = 81, -3          # past the table's row; below 0
    _, _, flags = run_attend(lib, (k, v, q, table, lens), dtype, kv_dtype)
    assert flags == llmq.LLMQ_PAGED_BAD_PAGE | llmq.LLMQ_PAGED_BAD_LEN
    seqs = torch.tensor([5, 5, -1, 6, 2 ** 30, 5], dtype=torch.int32, device="cuda")
    lens = torch.tensor([64, 3, 9, 9, 9, 30], dtype=torch.int32, device="cuda")
    _, _, flags = run_attend(lib, (k, v, q, table, lens), dtype, kv_dtype, seqs=seqs)
    assert flags == llmq.LLMQ_PAGED_BAD_LEN


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
def test_attention_large_scores(lib, dtype, kv_dtype):
    """Scores of hundreds, where an unshifted exponential overflows, and a scale given."""
    k, v, q, table, lens = attend_state([3, 200, 65], 8, 2, 64, 16, dtype, kv_dtype)
    run_attend(lib, (k, v, q * 30, table, lens), dtype, kv_dtype, scale=0.5)
    run_attend(lib, (k, v, q * 0, table, lens), dtype, kv_dtype)


@gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e20])
def test_attention_f32_queries_of_any_size_over_16_bits(lib, kv_dtype, size):
    """An f32 query keeps its range over a 16-bit pool: the scale undoes it."""
    k, v, q, table, lens = attend_state([7, 100], 8, 2, 64, 16, "f32", kv_dtype)
    run_attend(lib, (k, v, q * size, table, lens), "f32", kv_dtype, scale=0.125 / size)


@gpu
def test_attention_rows_of_one_sequence(lib):
    """Several rows read one table row at their own lengths (a prompt's rows)."""
    import torch
    k, v, q, table, lens = attend_state([90, 40], 8, 2, 64, 16, "f32", "f32")
    q = torch.randn((50, 8, 64), device="cuda")
    seqs = torch.tensor([0] * 30 + [1] * 20, dtype=torch.int32, device="cuda")
    lens = torch.tensor(list(range(61, 91)) + list(range(21, 41)), dtype=torch.int32, device="cuda")
    run_attend(lib, (k, v, q, table, lens), "f32", "f32", seqs=seqs)


@gpu
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_strided_rows_and_rows_behind(lib, dtype, kv_dtype):
    """q and out inside wider rows, not on 16 bytes; what lies between is left alone."""
    import torch
    k, v, q, table, lens = attend_state([9, 77, 130], 4, 2, 64, 16, dtype, kv_dtype)
    wide = torch.full((5, 300), 5.0, device="cuda").to(q.dtype)
    qs = wide.clone()
    qs[:3, 3:259] = q.view(3, 256)
    qv, ov = qs[:3, 3:259].unflatten(1, (4, 64)), wide[:3, 1:257].unflatten(1, (4, 64))
    lse = torch.full((5, 4), 5.0, device="cuda")
    a, work = attend_descriptor(lib, k, qv, ov, table, lens, dtype, lse=lse)
    kv = describe_pool(k, v, kv_dtype)
    ok(lib, lib.llmq_paged_attention(C.byref(kv), C.byref(a), None))
    torch.cuda.synchronize()
    check_attend(ov, lse[:3], attend_plain(k, v, q, table, lens), dtype, kv_dtype)
    assert (wide[3:] == 5).all() and (wide[:, :1] == 5).all() and (wide[:, 257:] == 5).all() and (lse[3:] == 5).all()


@gpu
@pytest.mark.parametrize("kv_dtype", ["f32", "bf16"])
def test_attention_offsets_past_32_bits(lib, kv_dtype):
    """Pages whose first element lies past 2^32 elements of the pool."""
    import torch
    n_pages = 40000  # of 16 x 8 x 1024 elements apart: 2^17 each
    stride = 1 << 17
    raw = torch.empty(n_pages * stride if kv_dtype == "bf16" else n_pages * stride, dtype=torch_type(kv_dtype),
                      device="cuda")
    pool = raw.view(n_pages, stride)[:, :16 * 2 * 64].unflatten(1, (16, 2, 64))
    used = torch.tensor([39999, 0, 33000, 32768, 16384, 39000], device="cuda")
    pool[used] = torch.randn((6, 16, 2, 64), device="cuda").to(pool.dtype)
    q = torch.randn((1, 8, 64), device="cuda")
    table, lens = used[None].int().contiguous(), torch.tensor([91], dtype=torch.int32, device="cuda")
    out, lse, flags = attend_gpu(lib, pool, pool, kv_dtype, q, table, lens, "f32")
    small = pool[used].clone()
    want = attend_plain(small, small, q, torch.arange(6)[None].int(), lens)
    check_attend(out, lse, want, "f32", kv_dtype)
    assert flags == 0


@gpu
def test_attention_same_bits_again_and_on_other_streams(lib):
    import torch
    st = attend_state([2000, 3, 901, 0, 77], 8, 2, 128, 16, "bf16", "bf16")
    k, v, q, table, lens = st
    first = attend_gpu(lib, k, v, "bf16", q, table, lens, "bf16")
    side = torch.cuda.Stream()
    for stream in (None, side, side):
        out, lse, _ = attend_gpu(lib, k, v, "bf16", q, table, lens, "bf16", stream=stream)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@gpu
@pytest.mark.parametrize("page", [2, 3, 8, 11, 40, 100, 129, 1000, 4097])
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("f16", "f16")])
def test_attention_page_sizes(lib, page, dtype, kv_dtype):
    run_attend(lib, attend_state([1, 130, 1003], 4, 2, 64, page, dtype, kv_dtype), dtype, kv_dtype)


@gpu
def test_attention_more_rows_than_a_launch_takes(lib):
    """1500 rows go in two launches that share the workspace."""
    import torch
    k, v, q, table, lens = attend_state([70, 33, 0, 129], 4, 2, 64, 16, "f32", "f32")
    g = torch.Generator().manual_seed(4)
    q = torch.randn((1500, 4, 64), generator=g).cuda()
    seqs = (torch.arange(1500) % 4).to(torch.int32).cuda()
    lens = (torch.arange(1500) % 70).to(torch.int32).cuda().clamp(max=lens[seqs.long()])
    run_attend(lib, (k, v, q, table, lens), "f32", "f32", seqs=seqs)


@gpu
def test_calls_of_two_threads_at_once(lib):
    """Each thread on its own stream with its own buffers: the results of calls one by one."""
    import threading

    import torch
    states = [attend_state([300, 7, 1200], 8, 2, 128, 16, *t) + (t,) for t in (("bf16", "bf16"), ("f32", "f32"))]
    want = [attend_gpu(lib, k, v, t[1], q, table, lens, t[0]) for k, v, q, table, lens, t in states]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        k, v, q, table, lens, t = states[i]
        st = torch.cuda.Stream()
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        kv = describe_pool(k, v, t[1])
        a, w = attend_descriptor(lib, k, q, out, table, lens, t[0], lse=lse)
        torch.cuda.synchronize()
        for _ in range(50):
            if lib.llmq_paged_attention(C.byref(kv), C.byref(a), st.cuda_stream) != 0:
                bad.append("error")
        st.synchronize()
        if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])):
            bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@gpu
def test_host_memory_is_refused(lib):
    import torch
    k, v, q, table, lens = attend_state([9, 77], 4, 2, 64, 16, "f32", "f32")
    out = torch.empty_like(q)
    for bad in ("lens", "table", "q"):
        for pinned in (False, True):
            d = dict(lens=lens, table=table, q=q)
            d[bad] = d[bad].cpu().pin_memory() if pinned else d[bad].cpu()
            a, work = attend_descriptor(lib, k, d["q"], out, d["table"], d["lens"], "f32")
            kv = describe_pool(k, v, "f32")
            refused(lib, lib.llmq_paged_attention, kv, a)


# ---------------------------------------------------------------- together
@gpu
@pytest.mark.parametrize("dtype,kv_dtype", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
def test_steps_in_a_captured_graph(lib, dtype, kv_dtype):
    """plan, append and attention captured once and replayed over several steps, the
    lengths and the free pages advanced on the GPU; two graphs share the
    workspace and replay one after the other.  Each step's output equals the
    plain form over everything appended so far."""
    import torch
    B, H, KV, hd, page, width, cap = 5, 8, 2, 64, 4, 8, 12
    i32 = dict(dtype=torch.int32, device="cuda")
    k, v = make_pool(B * width + 1, page, KV, hd, kv_dtype, fill=0.0)
    lens, head = torch.zeros(B, **i32), torch.zeros(1, **i32)
    added, table = torch.zeros(B, **i32), torch.full((B, width), -1, **i32)
    free = torch.randperm(B * width + 1, device="cuda").to(torch.int32)
    first, slots = torch.zeros(B + 1, **i32), torch.zeros(cap, dtype=torch.int64, device="cuda")
    pos, seqs, spans = (torch.zeros(cap, **i32) for _ in range(3))
    status = torch.zeros(1, **i32)
    t = torch_type(dtype)
    qkv = torch.zeros((cap, (H + 2 * KV) * hd), dtype=t, device="cuda")
    q, out = torch.zeros((cap, H, hd), dtype=t, device="cuda"), torch.zeros((cap, H, hd), dtype=t, device="cuda")
    lse = torch.zeros((cap, H), device="cuda")
    ang = torch.rand((64, hd // 2)) * 6
    cos, sin = torch.cos(ang).cuda().contiguous(), torch.sin(ang).cuda().contiguous()
    plan = llmq.PagedPlan(n_seqs=B, page_size=page, max_pages=width, max_rows=cap, n_free=free.numel(),
                          cached=ptr(lens), added=ptr(added), free_pages=ptr(free), free_head=ptr(head),
                          table=ptr(table), table_stride=width, lens=ptr(lens), first=ptr(first), slots=ptr(slots),
                          positions=ptr(pos), seqs=ptr(seqs), spans=ptr(spans), next_head=ptr(head),
                          status=ptr(status))
    kv = describe_pool(k, v, kv_dtype)
    e = qkv.element_size()
    app = llmq.PagedAppend(n_rows=cap, n_heads=H, dtype=CODES[dtype], rope_len=64, q=ptr(qkv), k=ptr(qkv) + H * hd * e,
                           v=ptr(qkv) + (H + KV) * hd * e, q_stride=qkv.stride(0), k_stride=qkv.stride(0),
                           v_stride=qkv.stride(0), q_out=ptr(q), q_out_stride=q.stride(0), slots=ptr(slots),
                           positions=ptr(pos), rope_cos=ptr(cos), rope_sin=ptr(sin), status=ptr(status))
    att, work = attend_descriptor(lib, k, q, out, table, spans, dtype, lse=lse, seqs=seqs, status=status)

    def step(st):
        ok(lib, lib.llmq_paged_plan(C.byref(plan), st))
        ok(lib, lib.llmq_paged_append(C.byref(kv), C.byref(app), st))
        ok(lib, lib.llmq_paged_attention(C.byref(kv), C.byref(att), st))

    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    torch.cuda.synchronize()
    assert lens.tolist() == [0] * B
    rng = np.random.default_rng(5)
    total = np.zeros(B, int)
    for i, add in enumerate([[3, 0, 1, 4, 2], [1, 1, 1, 1, 1], [0, 5, 1, 0, 1], [1, 1, 0, 1, 1], [0, 0, 0, 0, 0],
                             [2, 2, 2, 2, 2]]):
        added.copy_(torch.tensor(add, **i32))
        qkv.copy_(torch.tensor(rng.standard_normal(qkv.shape), dtype=t))
        out.fill_(9.0)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        total += add
        n = sum(add)
        assert lens.tolist() == total.tolist() and int(status) == 0 and int(head) == sum(-(-x // page) for x in total)
        s = dict(qkv=qkv, n_kv=KV, heads=H, hd=hd, k=k, v=v, q_out=q, cos=cos, sin=sin, slots=slots, positions=pos)
        check_append(s, append_plain(s))
        check_attend(out, lse, attend_plain(k, v, q, table, spans, seqs=seqs.cpu()), dtype, kv_dtype)
        assert (out[n:] == 0).all() and sorted(set(seqs[:n].tolist())) == [b for b in range(B) if add[b]]
