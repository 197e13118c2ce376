"""What the serving operators refuse before they look for a GPU, beside what their own tests
list: arrays that do not start on an element, where a load would fault."""
from __future__ import annotations

import ctypes as C

import pytest

import llmq
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
