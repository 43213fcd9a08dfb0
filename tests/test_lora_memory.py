"""Rows and outputs of the adapter projection that share memory: refused where a
CTA could store what another still reads, allowed where nothing is shared."""

import pytest
import torch

from test_lora_ops import check, make
from sglang_legolink_b200 import ops

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 300])
def test_outputs_that_share_memory_are_refused(M):
    t = make(M, 512, 512, 16, 3, "mixed", seed=M, device="cuda")
    stack, plan = ops.LoraStack(t["a"], t["b"], t["scale"]), ops.lora_plan(t["ids"], "cuda")
    call = lambda out, x=t["x"]: ops.linear_lora(x, t["w"], t["bias"], stack, plan, out=out)  # noqa: E731
    wide = torch.zeros(M + 1, 1040, dtype=BF, device="cuda")
    bad = [(t["x"], t["x"]), (wide[:M, 8:520], wide[:M, 512:1024]), (wide[:M, 512:1024], wide[:M, 8:520])]
    if M > 1:
        bad += [(torch.zeros(512, dtype=BF, device="cuda").expand(M, 512), t["x"]),
                (torch.zeros(M * 64 + 512, dtype=BF, device="cuda").as_strided((M, 512), (64, 1)), t["x"]),
                (t["w"][1:M + 1] if M < 511 else t["w"], t["x"])]
    for out, x in bad:
        with pytest.raises(RuntimeError, match="share"):
            call(out, x)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 300])
@pytest.mark.parametrize("xc,oc", [(0, 512), (512, 0), (0, 528), (528, 8)])
def test_columns_side_by_side_are_not(M, xc, oc):
    t = make(M, 512, 512, 16, 3, "mixed", seed=M, device="cuda")
    wide = torch.zeros(M, 1048, dtype=BF, device="cuda")
    wide[:, xc:xc + 512] = t["x"]
    t["x"] = wide[:, xc:xc + 512]
    check(t, out=wide[:, oc:oc + 512])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_one_vector_as_every_row(M):
    """Rows that all are one vector (stride 0): with each row's own adapter."""
    t = make(M, 512, 512, 16, 3, "mixed", seed=M, device="cuda")
    t["x"] = t["x"][:1].clone().expand(M, 512)
    check(t)
