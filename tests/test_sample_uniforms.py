"""Uniform numbers outside [0, 1), and none at all (NaN): the first and the last
kept token, in the statement and in the kernel."""

import pytest
import torch

from sglang_legolink_b200 import ops

NAN, INF = float("nan"), float("inf")


def case():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(7, 3000, generator=g) * 3
    x[:, :20] = -30.0  # none of the first tokens is kept
    u = torch.tensor([NAN, -1.0, -INF, 0.0, 1.0, 2.0, INF], dtype=torch.float64)
    return x, u, torch.ones(7), torch.full((7,), 40, dtype=torch.int32), torch.full((7,), 0.9)


def check(ids, logp, x, t, k, p):
    """The ends of what is kept, found with u at the middle of each token's share."""
    probe = torch.linspace(0, 1, 4001, dtype=torch.float64)[:-1] + 1 / 8000
    for b in range(7):
        row = x[b:b + 1].expand(4000, -1)
        seen = ops.sample(row, probe, t[:1].expand(4000), k[:1].expand(4000), p[:1].expand(4000))
        want = int(seen.min()) if b < 4 else int(seen.max())
        assert int(ids[b]) == want and float(logp[b]) > -INF


def test_the_statement():
    x, u, t, k, p = case()
    check(*ops.sample(x, u, t, k, p, return_logprobs=True), x, t, k, p)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [40, 2000])
def test_the_kernel(top):
    x, u, t, k, p = case()
    k[:] = top
    want, wlogp = ops.sample(x, u, t, k, p, return_logprobs=True)
    ids, logp = ops.sample(*(v.cuda() for v in (x, u, t, k, p)), return_logprobs=True)
    assert torch.equal(ids.cpu(), want) and bool(torch.isfinite(logp).all())
