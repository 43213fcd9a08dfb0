"""Rows of zeros and negative subnormals: the selection's ranges of keys end
between them, where -0 would be."""

import numpy as np
import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.ops import reference as ref


def key(x):
    """Order-preserving key of an fp32 value; -0 and +0 share one."""
    b = int(np.float32(x).view(np.uint32))
    b = 0 if b == 0x80000000 else b
    return b ^ 0xFFFFFFFF if b >> 31 else b | 0x80000000


def value(k):
    return np.uint32(k & 0x7FFFFFFF if k >> 31 else k ^ 0xFFFFFFFF).view(np.float32)


def last_value(hi):
    """Largest value that a range of keys ending with ``hi`` takes in."""
    return value(hi - 1 if hi == key(0.0) - 1 else hi)


def test_a_range_of_keys_takes_in_only_values_with_those_keys():
    tiny = value(key(0.0) - 2)  # the largest value below 0
    assert tiny < 0 and key(tiny) == key(0.0) - 2 and float(value(key(0.0) - 1)) == 0.0
    assert np.float32(0.0) <= value(0x7FFFFFFF)  # -0: the plain value of the end would take in 0, whose key is behind it
    for lo, hi in ((0x7FF00000, 0x7FFFFFFF), (0x7FFFFE00, 0x7FFFFFFF), (0x00800000, 0x80000000), (0x7FF00000, 0x80000005)):
        for x in (0.0, -0.0, tiny, value(lo), value(hi), value(lo + 1), value(0x80000001)):
            assert (value(lo) <= x <= last_value(hi)) <= (lo <= key(x) <= hi)


def rows(dtype, V, zeros, seed):
    """``zeros`` zeros (of either sign) among distinct negative subnormals."""
    g = torch.Generator().manual_seed(seed)
    bits = 23 if dtype == torch.float32 else 7
    out = []
    for _ in range(4):
        m = torch.randint(1, 1 << bits, (V,), generator=g)
        m[torch.randperm(V, generator=g)[:zeros]] = 0
        m |= (torch.rand(V, generator=g) < 0.5).long() * (m == 0) << (bits + 8)
        m |= (m != 0).long() << (bits + 8)
        out.append(m)
    m = torch.stack(out)
    if dtype == torch.float32:
        return (m - ((m >> 31) << 32)).to(torch.int32).view(torch.float32)
    return (m - ((m >> 15) << 16)).to(torch.int16).view(torch.bfloat16)


def test_the_rows_are_what_they_say():
    for dtype in (torch.float32, torch.bfloat16):
        x = rows(dtype, 3000, 200, 1)
        assert bool((x <= 0).all()) and bool((x.double().abs() < 2.0 ** -126).all()) and int((x == 0).sum()) == 4 * 200


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1.0, 1e38])  # with the second the search starts at the lowest key
@pytest.mark.parametrize("V,zeros", [(3000, 200), (60000, 5000)])
def test_the_cut_among_negative_subnormals_beside_zeros(V, zeros, T, dtype):
    x = rows(dtype, V, zeros, seed=V).cuda()
    u = torch.rand(4, generator=torch.Generator().manual_seed(2), dtype=torch.float64).cuda()
    t = torch.full((4,), T, device="cuda")
    for k, p in ((V // 2, None), (None, 0.5), (V - 7, 0.9), (None, 0.999)):
        kk = None if k is None else torch.full((4,), k, dtype=torch.int32, device="cuda")
        pp = None if p is None else torch.full((4,), p, device="cuda")
        want, _ = ref.sample(x, u, t, kk, pp)
        assert torch.equal(ops.sample(x, u, t, kk, pp), want), (k, p)
