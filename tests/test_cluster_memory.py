"""Distributed shared memory may be accessed only once every CTA of the cluster
has started, which a cluster barrier says.  A run cannot show that it is
missing (the other CTAs have nearly always started), the source can."""

import re
from pathlib import Path

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.ops import reference as ref

CSRC = Path(ops.__file__).resolve().parents[1] / "csrc"
REMOTE = re.compile(r"map_shared_rank\(|mapa\w*\(|ld_cluster\w*\(")
BARRIER = re.compile(r"barrier_wait\(|cluster_sync\(\)|cluster\.sync\(\)")


def kernels(path):
    """(name, body) of every __global__ function, without its comments."""
    src = re.sub(r"//[^\n]*", "", path.read_text())
    for m in re.finditer(r"__global__", src):
        at = src.index("{", m.end())
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(src[end], 0)
            end += 1
        yield re.findall(r"(\w+)\s*\(", src[m.end():at])[-1], src[at:end]


@pytest.mark.parametrize("file", sorted(p.name for p in CSRC.glob("*.cu")))
def test_a_cluster_barrier_comes_before_the_first_remote_access(file):
    for name, body in kernels(CSRC / file):
        remote = REMOTE.search(body)
        if remote:
            barrier = BARRIER.search(body)
            assert barrier and barrier.start() < remote.start(), f"{file}: {name}"


def test_the_search_sees_the_kernels_with_clusters():
    found = {n for p in CSRC.glob("*.cu") for n, body in kernels(p) if REMOTE.search(body)}
    assert {"sample_kernel", "lora_low_kernel", "lora_gemv_kernel"} <= found


@pytest.mark.gpu
def test_rows_of_many_ctas_launched_back_to_back_on_two_streams():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(3, 152064, generator=g, device="cuda") * 3).to(torch.bfloat16)
    u = torch.rand(3, generator=g, dtype=torch.float64, device="cuda")
    p = torch.tensor([0.9, 0.5, 1.0], device="cuda")
    want, _ = ref.sample(x, u, None, None, p)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(50):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.sample(x, u, None, None, p))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got)
