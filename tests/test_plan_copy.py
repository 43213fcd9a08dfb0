"""The engine makes a batch's adapter plan without waiting for the GPU."""

import numpy as np
import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import QwenModel
from sglang_legolink_b200.runtime.engine import Engine


def test_a_plan_goes_through_the_callers_copy():
    calls = []

    def copy(a):
        calls.append(a.copy())
        return torch.from_numpy(a.copy())

    p, q = ops.lora_plan([1, -1, 0, 1], "cpu", 3, copy), ops.lora_plan([1, -1, 0, 1], "cpu", 3)
    buf = p.buf
    assert len(calls) == 1 and torch.equal(p.buf, q.buf)
    p.update([2, 2, -1, 0]), q.update([2, 2, -1, 0])
    assert len(calls) == 2 and p.buf is buf and torch.equal(p.buf, q.buf)
    assert p.row_adapters.tolist() == [2, 2, -1, 0]


def test_a_plan_does_not_share_the_hosts_memory():
    ids = np.array([0, 1, 1], dtype=np.int64)
    p = ops.lora_plan(ids, "cpu")
    want = p.buf.clone()
    ids[:] = 7
    assert torch.equal(p.buf, want)


@pytest.mark.gpu
def test_the_engines_plans_do_not_wait():
    m = QwenModel.random_init(PRESETS["small-qwen2"], seed=0, device="cuda", dtype=torch.bfloat16)
    eng = Engine(m, num_pages=64, page_size=16, legolink_only=False)
    a, counts, n = [0, -1, 1], [200, 90, 14], 8
    first = eng._rows_plan(a, counts, n)  # allocates the staging buffer
    torch.cuda.synchronize()
    x = torch.randn(4096, 4096, device="cuda")
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            x = (x @ x).clamp(-1, 1)  # work ahead of the copies
        plan = eng._rows_plan(a, counts, n)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.set_sync_debug_mode("error")
    try:
        plan.update([1] * 304)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    again = ops.lora_plan([1] * 304, "cuda", n)
    assert torch.equal(plan.buf, again.buf)
    assert torch.equal(first.buf, ops.lora_plan(np.repeat(a, counts), "cuda", n).buf)
