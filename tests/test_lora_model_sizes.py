"""The adapter projection at the models' own depths (K to 25600, where the
few-row kernel's warps go round their registers more than once), at the borders
between its kernels, and what a row's result may depend on."""

import pytest
import torch

from test_lora_ops import check, formula64, make
from sglang_legolink_b200 import ops

SIZES = [  # M, K, N, R, adapters, rows: warps to a row and rank, CTAs of the few-row kernel
    (1, 18944, 3584, 16, 1, "all"),  # 8, 16: the down projection of Qwen2.5-7B
    (16, 18944, 3584, 16, 4, "mixed"),  # 8, 256
    (5, 18944, 3584, 40, 3, "mixed"),  # 8, 200
    (4, 25600, 5120, 32, 4, "all"),  # 8, 128: of Qwen3-32B
    (3, 16384, 512, 16, 3, "all"),  # the registers once, exactly
    (3, 16392, 512, 16, 3, "all"),  # and one vector more
    (7, 32776, 256, 8, 2, "mixed"),  # three times
    (2, 8192, 5120, 16, 2, "all"),  # 4, 16: the o projection of Qwen3-32B
    (3, 4104, 1024, 24, 2, "mixed"),  # 4
    (61, 8192, 1024, 16, 32, "mixed"),  # 4, 488 with many planes
    (37, 18944, 512, 16, 30, "mixed"),  # 8, 592
    (50, 2048, 1024, 64, 30, "mixed"),  # 1, 400
    (300, 1024, 512, 8, 20, "mixed"),  # 1, 300 in two tiles of rows
    (24, 18944, 1024, 128, 4, "mixed"),  # too many: tensor cores over a long K
    (600, 18944, 1024, 16, 6, "runs"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,K,N,R,n,rows", SIZES)
def test_against_64_bits(M, K, N, R, n, rows, swiglu):
    check(make(M, K, N, R, n, rows, seed=M + K, device="cuda"), swiglu)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n", [(32, 3584, 4608, 48, 20), (300, 512, 1024, 16, 40), (48, 3584, 1024, 32, 40),
                                       (64, 3584, 4608, 16, 64), (128, 1024, 512, 64, 100)])
def test_other_adapters_and_the_plans_capacity_change_a_row_by_rounding_alone(M, K, N, R, n):
    """The kernels and the splits of K go by the plan, so a row's sums may be
    taken in another order: within the bound of its formula, each way."""
    t = make(M, K, N, R, n, "mixed", seed=M, device="cuda")
    stack = ops.LoraStack(t["a"], t["b"], t["scale"])
    many = t["ids"].clone()
    many[7] = 3
    few = torch.full_like(many, -1)
    few[7] = 3
    got = []
    for ids in (many, few):
        want, tol = formula64({**t, "ids": ids}, False)
        exact = ops.lora_plan(ids, "cuda")
        for capacity in (exact.max_planes, max(32, M)):
            plan = ops.lora_plan(ids, "cuda", capacity)
            y = ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan)
            assert bool(((y.cpu().double() - want).abs() <= tol).all()), (capacity, ids is many)
            # and always in the same one for the same plan
            assert torch.equal(y, ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan))
            got.append(y[7].cpu().double())
    assert all(bool(((g - got[0]).abs() <= 2 * tol[7]).all()) for g in got)
    assert ops.check_errors("cuda") == 0


@pytest.mark.gpu
def test_a_bucket_of_32_in_a_graph_equals_the_same_plan_outside_it():
    """Many adapters in a captured decode, its plan updated between replays:
    bit for bit the eager forward with a plan of the graph's capacity."""
    from test_adapters import engine, gpu_seqs
    from sglang_legolink_b200.models.qwen import ForwardBatch

    eng, ads = engine("small-qwen2", "cuda", torch.bfloat16)
    from test_adapters import state_of
    from sglang_legolink_b200.models.adapters import Adapter

    for i in range(10):
        eng.load_adapter(f"more{i}", Adapter.from_state(state_of(eng.cfg, 8, 50 + i, ("q_proj", "o_proj", "down_proj")), 16, 8))
    names = [None, *eng.adapters]
    bucket = 32
    for shift in range(3):
        seqs = gpu_seqs(eng, [names[(i * (shift + 1) + shift) % len(names)] for i in range(29)], n=20)
        for _ in range(2):
            for s in seqs:
                eng._ensure_capacity(s, s.length + 1)
            ids, pos, slots, pt, kvl = eng._decode_inputs(seqs, bucket, -(-eng.max_context // 16))
            plan = eng._rows_plan([s.adapter for s in seqs] + [-1] * (bucket - len(seqs)), 1, bucket)
            fb = ForwardBatch(mode="decode", input_ids=ids.cuda(), positions=pos.cuda(), slots=slots.cuda(),
                              q_indptr=torch.arange(bucket + 1, dtype=torch.int32).cuda(), page_table=pt.cuda(),
                              kv_lens=kvl.cuda(), logit_rows=None, lora=plan,
                              decode_nsplit=ops.decode_splits(bucket, eng.model.hkv, eng.max_context))
            want = eng.model.forward(fb, eng.kv)[: len(seqs)].clone()
            out = eng.decode_step(seqs)
            assert torch.equal(eng._graphs[("adapters", bucket)]["logits"][: len(seqs)], want)
            for s, t in zip(seqs, out):
                s.output_ids.append(t)
        for s in seqs:
            eng.free(s)
