"""What the serving operators refuse before they look for a GPU, beside what their own tests
list: arrays that do not start on an element, where a load would fault, and counts whose
indices would not fit 31 bits."""
from __future__ import annotations

import ctypes as C

import pytest

import llmq
from conftest import has_gpu
from test_paged import F, append_args, attend_args, plan_args, pool_args, refused
from test_sample_rows import args as sample_args

PLAN = "cached added free_pages free_head table lens first slots positions seqs spans next_head status".split()
APPEND = "slots positions rope_cos rope_sin status".split()
ATTEND = "lse table seqs lens status".split()
SAMPLE = "temperature top_k top_p min_p u ids logprobs".split()


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("call,name", [("plan", n) for n in PLAN] + [("append", n) for n in APPEND] +
                         [("attend", n) for n in ATTEND] + [("sample", n) for n in SAMPLE])
def test_arrays_off_their_elements(lib, call, name, off):
    bad = {name: F + off}
    if call == "plan":
        refused(lib, lib.llmq_paged_plan, plan_args(**bad))
    elif call == "append":
        refused(lib, lib.llmq_paged_append, pool_args(), append_args(**bad))
    elif call == "attend":
        refused(lib, lib.llmq_paged_attention, pool_args(), attend_args(**bad))
    else:
        refused(lib, lib.llmq_sample_rows, sample_args(**bad))


def test_slots_are_64_bit(lib):
    refused(lib, lib.llmq_paged_plan, plan_args(slots=F + 4))
    refused(lib, lib.llmq_paged_append, pool_args(), append_args(slots=F + 4))


MOST = 2**31 - 1 - 4096


@pytest.mark.skipif(has_gpu(), reason="this machine has a GPU, whose memory the good calls do not name")
def test_counts_up_to_the_limits_pass_the_checks(lib):
    for rc in (lib.llmq_paged_plan(C.byref(plan_args(n_seqs=MOST)), None),
               lib.llmq_paged_append(C.byref(pool_args()), C.byref(append_args(n_rows=MOST)), None),
               lib.llmq_paged_attention(C.byref(pool_args()), C.byref(attend_args(n_rows=MOST, seqs=F)), None)):
        assert rc == llmq.LLMQ_ERR_NO_DEVICE
    lib.q_llama_clear_error()


@pytest.mark.parametrize("n", [MOST + 1, 2**31 - 1])
def test_counts_past_31_bit_indices(lib, n):
    refused(lib, lib.llmq_paged_plan, plan_args(n_seqs=n))
    refused(lib, lib.llmq_paged_append, pool_args(), append_args(n_rows=n))
    refused(lib, lib.llmq_paged_attention, pool_args(), attend_args(n_rows=n, seqs=F))


def test_rows_past_31_bit_indices(lib):
    wide = dict(n_heads=1 << 25, q_stride=1 << 31)
    refused(lib, lib.llmq_paged_append, pool_args(), append_args(q_out_stride=1 << 31, **wide))
    refused(lib, lib.llmq_paged_attention, pool_args(), attend_args(out_stride=1 << 31, **wide))
