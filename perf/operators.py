"""The serving operators as they are measured: block tables and slot maps, the
paged cache's writer, attention of one new token over a paged cache, and
sampling of a batch of logits rows.

Plain forms are elementary torch operations in 32 bits (64 for the sampler,
whose choices lie at borders of long sums).  With `own` set, `run` calls
libllmq_cuda.so through its Python binding.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 requests, as the 8B serving workload runs it
        dict(name="plan_decode_64", op="plan", seqs=64, page=16, lo=2048, hi=2176, prompts=0, prompt_hi=1),
        # a full scheduler queue: mostly decoding requests, some prompts entering
        dict(name="plan_mixed_1000", op="plan", seqs=1000, page=24, lo=0, hi=2176, prompts=200, prompt_hi=1030),
        # one token of the tiny model: latency
        dict(name="append_tiny_1", op="append", tokens=1, heads=6, kv=2, hd=48, page=16, dtype="f32", kv_dtype="f32",
             max_pos=256),
        # a batched step of the 8B shape whose cache is kept in 16 bits
        dict(name="append_decode_64", op="append", tokens=64, heads=32, kv=8, hd=128, page=16, dtype="f32",
             kv_dtype="bf16", max_pos=2176),
        # prompts of the 8B shape, all in 16 bits
        dict(name="append_prompts_16384", op="append", tokens=16384, heads=32, kv=8, hd=128, page=64, dtype="bf16",
             kv_dtype="bf16", max_pos=2176),
        # one token of the tiny model at the end of its context: latency
        dict(name="attend_tiny_1", op="attend", rows=1, heads=6, kv=2, hd=48, page=16, dtype="f32", kv_dtype="f32",
             lo=256, hi=256, window=0),
        # the 8B serving step: 64 sequences at 2048 to 2176 cached positions, f32 cache
        dict(name="attend_8b_64_f32", op="attend", rows=64, heads=32, kv=8, hd=128, page=16, dtype="f32",
             kv_dtype="f32", lo=2048, hi=2176, window=0),
        # ragged lengths in 16 bits, page ends inside every tile
        dict(name="attend_ragged_61_bf16", op="attend", rows=61, heads=32, kv=8, hd=128, page=24, dtype="bf16",
             kv_dtype="bf16", lo=1, hi=8191, window=0),
        # one long sequence of the 70B shape: only its length can be split
        dict(name="attend_long_1_f16", op="attend", rows=1, heads=64, kv=8, hd=128, page=64, dtype="f16",
             kv_dtype="f16", lo=131071, hi=131071, window=0),
        # the command line's settings on one row of a 32000-word vocabulary: latency
        dict(name="sample_cli_1", op="sample", rows=1, vocab=32000, dtype="f32", kind="cli"),
        # a batch whose requests each have their own settings
        dict(name="sample_mixed_64", op="sample", rows=64, vocab=128256, dtype="f32", kind="mixed"),
        # a large batch without top-k: nucleus, min-p and plain sampling
        dict(name="sample_nucleus_256", op="sample", rows=256, vocab=128256, dtype="bf16", kind="nucleus"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "sample"])
    if op == "plan":
        seqs = _log_int(rng, 1, 1000)
        return dict(op=op, seqs=seqs, page=rng.choice([1, 8, 16, 24, 32, 64, 100, 128]), lo=0,
                    hi=_log_int(rng, 16, 2176), prompts=rng.randint(0, seqs // 5), prompt_hi=_log_int(rng, 1, 1030))
    if op == "append":
        kv = rng.choice([1, 2, 4, 8])
        dtype = rng.choice(["f32", "bf16", "f16"])
        kv_dtype = rng.choice(["f32", "bf16", "f16"]) if dtype == "f32" else dtype
        return dict(op=op, tokens=_log_int(rng, 1, 8000), heads=kv * rng.randint(1, 4), kv=kv,
                    hd=rng.choice([48, 64, 80, 96, 128]), page=rng.choice([1, 8, 16, 24, 32, 64]), dtype=dtype,
                    kv_dtype=kv_dtype, max_pos=rng.randint(64, 2176))
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8])
        hd = rng.choice([48, 64, 80, 96, 128])
        dtype = rng.choice(["f32", "bf16", "f16"])
        kv_dtype = rng.choice(["f32", "bf16", "f16"]) if dtype == "f32" else dtype
        rows = _log_int(rng, 1, 150)
        hi = _log_int(rng, 1, min(65536, 60000 * 8 // (rows * kv)))
        return dict(op=op, rows=rows, heads=kv * rng.choice([1, 2, 3, 4, 7, 8]), kv=kv, hd=hd,
                    page=rng.choice([8, 16, 24, 32, 64, 128]), dtype=dtype, kv_dtype=kv_dtype,
                    lo=rng.choice([0, 1, max(1, hi // 2), hi]), hi=hi,
                    window=rng.choice([0, 0, 0, _log_int(rng, 1, hi)]))
    return dict(op=op, rows=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 128256),
                dtype=rng.choice(["f32", "bf16", "f16"]), kind=rng.choice(["cli", "mixed", "nucleus"]))


def _lengths(case, n):
    """The case's n lengths: the same for every seed, whose permutation of them differs."""
    rng = random.Random("%d %d %d" % (n, case["lo"], case["hi"]))
    v = [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
    if n:
        v[0] = case["hi"]
    return v


def _plan_lengths(case):
    """(cached, added) of a plan's requests."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["hi"], case["prompts"]))
    cached = _lengths(case, case["seqs"])
    added = [1] * case["seqs"]
    for i in range(case["prompts"]):
        cached[i], added[i] = 0, rng.randint(1, case["prompt_hi"])
    return cached, added


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _tables(lens, page, g):
    """A pool's pages in random order: (table rows padded with -1, pages in the pool)."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + 5
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need))
    first = [0]
    for n in need:
        first.append(first[-1] + n)
    at = torch.tensor(first[:-1], device="cuda")[:, None] + torch.arange(width, device="cuda")[None, :]
    used = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, perm[at.clamp(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total


def _prepare_plan(case, seed):
    g = _gen(seed)
    cached, added = _plan_lengths(case)
    order = list(range(len(cached)))
    random.Random(seed).shuffle(order)
    cached, added = [cached[i] for i in order], [added[i] for i in order]
    page, n = case["page"], len(cached)
    have = [(c + page - 1) // page for c in cached]
    need = [(c + a + page - 1) // page for c, a in zip(cached, added)]
    total = sum(need) + 7
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(need) + 1
    first = [0]
    for h in have:
        first.append(first[-1] + h)
    at = torch.tensor(first[:-1], device="cuda")[:, None] + torch.arange(width, device="cuda")[None, :]
    used = torch.arange(width, device="cuda")[None, :] < torch.tensor(have, device="cuda")[:, None]
    table = torch.where(used, perm[at.clamp(max=total - 1)], -1).to(torch.int32).contiguous()
    rows = sum(added) + 3  # a step's rows are padded
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(case=case, page=page, width=width, rows=rows, cached=torch.tensor(cached, **i32),
                added=torch.tensor(added, **i32), table=table, free=perm[first[-1]:].contiguous(),
                head=torch.zeros(1, **i32), next_head=torch.zeros(1, **i32), lens=torch.zeros(n, **i32),
                first=torch.zeros(n + 1, **i32), slots=torch.zeros(rows, dtype=torch.int64, device="cuda"),
                positions=torch.zeros(rows, **i32), seqs=torch.zeros(rows, **i32), spans=torch.zeros(rows, **i32),
                status=torch.zeros(1, **i32))


def _prepare_append(case, seed):
    g = _gen(seed)
    T, H, KV, hd, page = case["tokens"], case["heads"], case["kv"], case["hd"], case["page"]
    t, kt = DTYPES[case["dtype"]], DTYPES[case["kv_dtype"]]
    pages = (T + page - 1) // page + 3
    # one packed row of q, k and v a token, as the QKV product leaves it
    qkv = torch.randn((T, (H + 2 * KV) * hd), generator=g, device="cuda").to(t)
    cache = torch.randn((2, pages, page, KV, hd), generator=g, device="cuda").to(kt)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].contiguous()
    pos = torch.randint(0, case["max_pos"], (T,), generator=g, device="cuda", dtype=torch.int32)
    ang = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) * 2 / hd)[None, :]
    return dict(case=case, qkv=qkv, k=cache[0], v=cache[1], slots=slots, positions=pos,
                cos=torch.cos(ang).float().contiguous(), sin=torch.sin(ang).float().contiguous(),
                q_out=torch.empty((T, H, hd), dtype=t, device="cuda"))


def _prepare_attend(case, seed):
    g = _gen(seed)
    R, H, KV, hd, page = case["rows"], case["heads"], case["kv"], case["hd"], case["page"]
    t, kt = DTYPES[case["dtype"]], DTYPES[case["kv_dtype"]]
    lens = _lengths(case, R)
    random.Random(seed).shuffle(lens)
    table, pages = _tables(lens, page, g)
    q = torch.randn((R, H, hd), generator=g, device="cuda").to(t)
    pool = torch.empty((2, pages, page, KV, hd), dtype=kt, device="cuda")
    pool.normal_(generator=g)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return dict(case=case, q=q, k=pool[0], v=pool[1], table=table, lens=lens,
                out=torch.empty((R, H, hd), dtype=t, device="cuda"),
                lse=torch.empty((R, H), dtype=torch.float32, device="cuda"))


def _prepare_sample(case, seed):
    g = _gen(seed)
    R, V = case["rows"], case["vocab"]
    # logits of a trained model: a smooth body and a few words that stand out
    logits = torch.randn((R, V), generator=g, device="cuda") * 2.0
    top = torch.randint(0, V, (R, 1), generator=g, device="cuda") + torch.arange(40, device="cuda") * (V // 40)
    top = top % V
    logits.scatter_(1, top, 4.0 + 4.0 * torch.rand((R, 40), generator=g, device="cuda"))
    logits = logits.to(DTYPES[case["dtype"]])
    rng = random.Random(seed)
    pick = {"cli": lambda: (0.8, 40, 0.95, 0.0),
            "mixed": lambda: rng.choice([(0.8, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 50, 1.0, 0.0),
                                         (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (1.2, 1000, 0.99, 0.01)]),
            "nucleus": lambda: rng.choice([(1.0, 0, 0.95, 0.0), (0.7, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.1),
                                           (1.0, 0, 1.0, 0.0)])}[case["kind"]]
    s = [pick() for _ in range(R)]
    f = dict(dtype=torch.float32, device="cuda")
    return dict(case=case, logits=logits, temperature=torch.tensor([x[0] for x in s], **f),
                top_k=torch.tensor([x[1] for x in s], dtype=torch.int32, device="cuda"),
                top_p=torch.tensor([x[2] for x in s], **f), min_p=torch.tensor([x[3] for x in s], **f),
                u=torch.rand(R, generator=g, device="cuda"),
                ids=torch.empty(R, dtype=torch.int32, device="cuda"), logprobs=torch.empty(R, **f))


def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["op"]](case, seed)


# ------------------------------------------------------------- plain forms
def _plain_plan(s):
    page, rows, width = s["page"], s["rows"], s["width"]
    cached, added = s["cached"].long(), s["added"].long()
    have, need = (cached + page - 1) // page, (cached + added + page - 1) // page
    new = need - have
    upto = torch.cumsum(new, 0)
    col = torch.arange(width, device="cuda")[None, :]
    at = s["head"].long() + (upto - new)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"])
    ends = torch.cumsum(added, 0)
    first = torch.cat([torch.zeros_like(ends[:1]), ends])
    r = torch.arange(rows, device="cuda")
    live = r < ends[-1]
    b = torch.searchsorted(ends, r, right=True).clamp(max=cached.numel() - 1)
    pos = cached[b] + r - first[b]
    slot = table[b, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    none = torch.full_like(pos, -1)
    return (table, (cached + added).int(), first.int(), torch.where(live, slot, none),
            torch.where(live, pos, none).int(), torch.where(live, b, none).int(),
            torch.where(live, pos + 1, none + 1).int(), (s["head"] + upto[-1:]).int())


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    T, H, KV, hd = c["tokens"], c["heads"], c["kv"], c["hd"]
    x = s["qkv"].view(T, H + 2 * KV, hd)
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    q = _rotate(x[:, :H].float(), cos, sin).to(x.dtype)
    k = _rotate(x[:, H:H + KV].float(), cos, sin).to(s["k"].dtype)
    s["k"].view(-1, KV, hd)[s["slots"]] = k
    s["v"].view(-1, KV, hd)[s["slots"]] = x[:, H + KV:].to(s["v"].dtype)
    return s["k"], s["v"], q


def _plain_attend(s):
    c = s["case"]
    R, H, KV, hd = c["rows"], c["heads"], c["kv"], c["hd"]
    G = H // KV
    at = s["table"].clamp(min=0).long()
    k = s["k"][at].view(R, -1, KV, hd).float().transpose(1, 2)  # [R, KV, L, hd]
    v = s["v"][at].view(R, -1, KV, hd).float().transpose(1, 2)
    L = k.shape[2]
    q = s["q"].float().view(R, KV, G, hd) * (1.0 / math.sqrt(hd))
    sc = q @ k.transpose(2, 3)
    p = torch.arange(L, device="cuda")[None, :]
    n = s["lens"].long()[:, None]
    seen = (p < n) & (p >= (n - c["window"] if c["window"] else 0 * n))
    sc = sc.masked_fill(~seen[:, None, None, :], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(sc - m)
    z = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(z > 0, z, torch.ones_like(z))
    lse = torch.where(z > 0, m + torch.log(z), torch.full_like(z, float("-inf")))
    return o.view(R, H, hd).to(s["q"].dtype), lse.view(R, H)


def _plain_sample(s):
    V = s["case"]["vocab"]
    l, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    T = s["temperature"].double()[:, None]
    d = (l.double() - l[:, :1].double()) / torch.where(T > 0, T, torch.ones_like(T))
    w = torch.exp(d)
    C = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(C[:, :1]), C[:, :-1]], 1)
    i = torch.arange(V, device="cuda")[None, :]
    k = s["top_k"].long()[:, None]
    p, mp = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    kept = ((k <= 0) | (i < k)) & (w >= mp) & ((p <= 0) | (p >= 1) | (before < p * C[:, -1:]))
    kept = kept & ((T > 0) | (i < 1))
    n = kept.sum(1, keepdim=True).clamp(min=1)
    z = torch.gather(C, 1, n - 1)
    at = (C < s["u"].double()[:, None] * z).sum(1, keepdim=True)
    at = torch.minimum(at, n - 1)
    ids = torch.gather(order, 1, at)[:, 0].int()
    return ids, torch.log(torch.gather(w, 1, at) / z)[:, 0].float()


# ------------------------------------------------- the library's own calls
def _lib():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "llm-project_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import llmq
    return llmq, llmq.load()


_CODES = {"f32": 0, "f16": 1, "bf16": 2}


def _paged_kv(llmq, s):
    c, k = s["case"], s["k"]
    return llmq.PagedKV(k=k.data_ptr(), v=s["v"].data_ptr(), dtype=_CODES[c["kv_dtype"]], n_pages=k.shape[0],
                        page_size=k.shape[1], n_kv=k.shape[2], head_dim=k.shape[3], page_stride=k.stride(0),
                        token_stride=k.stride(1), head_stride=k.stride(2))


def _describe(s):
    """The call's descriptors: pointers, sizes and strides, which a program fills once for the buffers it keeps."""
    llmq, lib = _lib()
    c = s["case"]
    if c["op"] == "plan":
        a = llmq.PagedPlan(n_seqs=c["seqs"], page_size=c["page"], max_pages=s["width"], max_rows=s["rows"],
                           n_free=s["free"].numel(), cached=s["cached"].data_ptr(), added=s["added"].data_ptr(),
                           free_pages=s["free"].data_ptr(), free_head=s["head"].data_ptr(),
                           table=s["table"].data_ptr(), table_stride=s["table"].stride(0), lens=s["lens"].data_ptr(),
                           first=s["first"].data_ptr(), slots=s["slots"].data_ptr(),
                           positions=s["positions"].data_ptr(), seqs=s["seqs"].data_ptr(),
                           spans=s["spans"].data_ptr(), next_head=s["next_head"].data_ptr(),
                           status=s["status"].data_ptr())
        outs = tuple(s[n] for n in ("table", "lens", "first", "slots", "positions", "seqs", "spans", "next_head"))
        return lib.llmq_paged_plan, (llmq.C.byref(a),), outs, lib
    if c["op"] == "append":
        H, KV, hd, x = c["heads"], c["kv"], c["hd"], s["qkv"]
        kv, e = _paged_kv(llmq, s), x.element_size()
        a = llmq.PagedAppend(n_rows=c["tokens"], n_heads=H, dtype=_CODES[c["dtype"]], rope_len=s["cos"].shape[0],
                             q=x.data_ptr(), k=x.data_ptr() + H * hd * e, v=x.data_ptr() + (H + KV) * hd * e,
                             q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0),
                             q_out=s["q_out"].data_ptr(), q_out_stride=s["q_out"].stride(0),
                             slots=s["slots"].data_ptr(), positions=s["positions"].data_ptr(),
                             rope_cos=s["cos"].data_ptr(), rope_sin=s["sin"].data_ptr())
        return lib.llmq_paged_append, (llmq.C.byref(kv), llmq.C.byref(a)), (s["k"], s["v"], s["q_out"]), lib
    if c["op"] == "attend":
        kv, q = _paged_kv(llmq, s), s["q"]
        size = lib.llmq_paged_attention_workspace(c["rows"], c["heads"], c["kv"], c["hd"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        a = llmq.PagedAttention(n_rows=c["rows"], n_heads=c["heads"], dtype=_CODES[c["dtype"]], window=c["window"],
                                max_pages=s["table"].shape[1], n_seqs=s["table"].shape[0], q=q.data_ptr(),
                                q_stride=q.stride(0), out=s["out"].data_ptr(), out_stride=s["out"].stride(0),
                                lse=s["lse"].data_ptr(), table=s["table"].data_ptr(),
                                table_stride=s["table"].stride(0), lens=s["lens"].data_ptr(),
                                workspace=s["workspace"].data_ptr(), workspace_bytes=size)
        return lib.llmq_paged_attention, (llmq.C.byref(kv), llmq.C.byref(a)), (s["out"], s["lse"]), lib
    a = llmq.SampleRows(n_rows=c["rows"], vocab=c["vocab"], dtype=_CODES[c["dtype"]], logits=s["logits"].data_ptr(),
                        stride=s["logits"].stride(0), temperature=s["temperature"].data_ptr(),
                        top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(), min_p=s["min_p"].data_ptr(),
                        u=s["u"].data_ptr(), ids=s["ids"].data_ptr(), logprobs=s["logprobs"].data_ptr())
    return lib.llmq_sample_rows, (llmq.C.byref(a),), (s["ids"], s["logprobs"]), lib


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _describe(state)
        fn, args, outs, lib = state["call"]
        if fn(*args, torch.cuda.current_stream().cuda_stream) != 0:
            raise RuntimeError(lib.q_llama_last_error_message().decode())
        return outs
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
            "sample": _plain_sample}[state["case"]["op"]](state)


# ------------------------------------------------------------- what it costs
def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    c = case
    if c["op"] == "plan":
        cached, added = _plan_lengths(c)
        page, rows = c["page"], sum(added)
        new = sum((a + b + page - 1) // page - (a + page - 1) // page for a, b in zip(cached, added))
        return {"bytes": 16 * c["seqs"] + 8 * new + 24 * rows, "flops": 4 * rows}
    if c["op"] == "append":
        T, H, KV, hd = c["tokens"], c["heads"], c["kv"], c["hd"]
        e, k = _bytes(c["dtype"]), _bytes(c["kv_dtype"])
        angles = min(T, c["max_pos"]) * hd * 4
        return {"bytes": T * (hd * ((2 * H + 2 * KV) * e + 2 * KV * k) + 12) + angles, "flops": 3 * T * (H + KV) * hd}
    if c["op"] == "attend":
        seen = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c, c["rows"]))
        per = c["rows"] * c["heads"] * (2 * c["hd"] * _bytes(c["dtype"]) + 4)
        return {"bytes": 2 * seen * c["kv"] * c["hd"] * _bytes(c["kv_dtype"]) + per,
                "flops": 4 * seen * c["heads"] * c["hd"]}
    return {"bytes": c["rows"] * (c["vocab"] * _bytes(c["dtype"]) + 28), "flops": 2 * c["rows"] * c["vocab"]}


# ------------------------------------------------------ 64 bits, written apart
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "append":
        H, KV, hd = case["heads"], case["kv"], case["hd"]
        half = hd // 2
        x = s["qkv"].double().reshape(case["tokens"], -1, hd)
        cos, sin = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
        turned = torch.empty_like(x[:, :H + KV])
        for d in range(half):
            a, b = x[:, :H + KV, d], x[:, :H + KV, d + half]
            turned[:, :, d] = a * cos[:, d:d + 1] - b * sin[:, d:d + 1]
            turned[:, :, d + half] = a * sin[:, d:d + 1] + b * cos[:, d:d + 1]
        k, v = s["k"].double().reshape(-1, KV, hd), s["v"].double().reshape(-1, KV, hd)
        k.index_copy_(0, s["slots"], turned[:, H:])
        v.index_copy_(0, s["slots"], x[:, H + KV:])
        return k.reshape(s["k"].shape), v.reshape(s["v"].shape), turned[:, :H].contiguous()
    if case["op"] == "attend":
        R, H, KV, hd, page = case["rows"], case["heads"], case["kv"], case["hd"], case["page"]
        o = torch.zeros((R, H, hd), dtype=torch.float64, device="cuda")
        lse = torch.full((R, H), float("-inf"), dtype=torch.float64, device="cuda")
        for r, n in enumerate(s["lens"].tolist()):
            a = max(0, n - case["window"]) if case["window"] else 0
            if n <= a:
                continue
            p = torch.arange(a, n, device="cuda")
            page_of = s["table"][r].long()[p // page]
            k, v = s["k"][page_of, p % page].double(), s["v"][page_of, p % page].double()
            for h in range(H):
                t = (k[:, h // (H // KV)] * s["q"][r, h].double()).sum(1) / hd ** 0.5
                lse[r, h] = torch.logsumexp(t, 0)
                o[r, h] = (torch.exp(t - lse[r, h])[:, None] * v[:, h // (H // KV)]).sum(0)
        return o, lse
    # the log probability of the id that the rules draw, row by row
    out = torch.zeros(case["rows"], dtype=torch.float64)
    lg = s["logits"].double().cpu()
    sets = [s[n].double().tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u")]
    for r, (T, k, p, mp, u) in enumerate(zip(*sets)):
        if not T > 0:
            continue
        w, _ = torch.sort(torch.exp((lg[r] - lg[r].max()) / T), descending=True)
        total, n = float(w.sum()), w.numel()
        n = min(n, int(k)) if k > 0 else n
        n = min(n, int((w >= mp).sum()))
        C = torch.cumsum(w, 0)
        if 0 < p < 1:
            n = min(n, int(torch.searchsorted(C, torch.tensor(p * total, dtype=torch.float64))) + 1)
        n = max(n, 1)
        i = min(int(torch.searchsorted(C, torch.tensor(u * float(C[n - 1]), dtype=torch.float64))), n - 1)
        out[r] = torch.log(w[i] / C[n - 1])
    return None, out
