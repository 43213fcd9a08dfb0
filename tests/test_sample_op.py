"""Drawing one token per row with temperature, top-k, top-p and min-p from
given uniform numbers: the statement against a token-by-token one here, the
kernel against the statement (float64) on a GPU."""

import math

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.ops import reference as ref

INF = float("inf")


def by_hand(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row, in Python floats."""
    x = [(-INF if math.isnan(v) else v) for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    top = x[order[0]]
    if top == -INF:
        return -1, -INF
    if not t > 0:
        return order[0], 0.0
    w = [1.0 if v == top else 0.0 if v == -INF or top == INF else math.exp((v - top) / t) for v in x]
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        total, run, n = math.fsum(w[i] for i in order), 0.0, 0
        while n < len(order) and (n == 0 or run < p * total):
            run += w[order[n]]
            n += 1
        order = order[:n]
    if m > 0:
        order = [i for i in order if w[i] >= min(m, 1.0)]
    total, run = math.fsum(w[i] for i in order), 0.0
    for i in sorted(order):
        run += w[i]
        if run > u * total:
            return i, math.log(w[i] / total)
    raise AssertionError


def settings(B, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)

    def pick(v):
        return torch.tensor(v)[torch.randint(0, len(v), (B,), generator=g)].to(device)

    return (torch.rand(B, generator=g, dtype=torch.float64).to(device), pick([0.0, 0.3, 0.7, 1.0, 2.5]),
            pick([0, -1, 1, 2, 20, 100, 100000]).to(torch.int32), pick([1.0, 0.1, 0.8, 0.95, 0.999, 0.0]),
            pick([0.0, 0.0, 0.02, 0.3, 1.0]))


def logits_of(kind, B, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 2
    if kind == "tail":
        x = x + 1.5 * torch.empty(B, V).exponential_(generator=g)
    elif kind == "coarse":  # many equal values
        x = x.round()
    elif kind == "equal":
        x = torch.full((B, V), -3.0)
    elif kind == "masked":
        x[torch.rand(B, V, generator=g) < 0.9] = -INF
        x[torch.rand(B, V, generator=g) < 0.02] = float("nan")
        x[0] = -INF
    elif kind == "lowest":  # masks of the type's lowest value
        x[torch.rand(B, V, generator=g) < 0.9] = torch.finfo(dtype).min
    elif kind == "infinite":
        x[torch.rand(B, V, generator=g) < 0.01] = INF
    elif kind == "wide":
        x = x * 1e4
    elif kind == "zeros":
        x = torch.where(torch.rand(B, V, generator=g) < 0.5, torch.tensor(-0.0), torch.tensor(0.0))
    return x.to(dtype)


KINDS = ["normal", "tail", "coarse", "equal", "masked", "lowest", "infinite", "wide", "zeros"]


# --------------------------------------------------------------------- CPU
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [1, 2, 37, 300])
def test_statement_by_hand(kind, V):
    B = 24
    x = logits_of(kind, B, V, seed=V)
    u, t, k, p, m = settings(B, seed=V + 1)
    ids, logp = ops.sample(x, u, t, k, p, m, return_logprobs=True)
    for b in range(B):
        i, lp = by_hand(x[b].double().tolist(), *(float(v[b]) for v in (u, t)), int(k[b]), float(p[b]), float(m[b]))
        assert int(ids[b]) == i, (b, kind)
        assert float(logp[b]) == pytest.approx(lp, abs=1e-5)


def test_defaults_and_frequencies():
    x = torch.tensor([[0.0, 1.0, 2.0]]).repeat(3000, 1)
    u = (torch.arange(3000, dtype=torch.float64) + 0.5) / 3000
    n = torch.bincount(ops.sample(x, u).long(), minlength=3).double() / 3000
    # a grid of u: each share is met within one grid step
    assert torch.allclose(n, torch.softmax(x[0].double(), 0), atol=1.1 / 3000)
    assert ops.sample(x[:0], u[:0]).shape == (0,)
    out = torch.empty(3000, dtype=torch.int32)
    assert ops.sample(x, u, out=out) is out
    with pytest.raises(ValueError):
        ops.sample(x[0], u)


# --------------------------------------------------------------------- GPU
def on_gpu(x, u, t=None, k=None, p=None, m=None):
    d = [None if v is None else v.cuda() for v in (t, k, p, m)]
    x = x if x.is_cuda else x.cuda()
    ids, logp = ops.sample(x, u.cuda(), *d, return_logprobs=True)
    want, wlogp = ref.sample(x, u.cuda(), *d)
    assert torch.equal(ids, want), (ids != want).nonzero()[:, 0].tolist()
    # Both round the log to fp32: one step of it apart at most.  The kernel has
    # each weight to 1.2e-12 < 2^-39 of itself (in the sum and in the token's
    # own) and both round the up to V weights to 2^-44, off by half of that;
    # the sum is then exact, and it is 1 or more.
    tol = 2.0 ** -23 * wlogp.abs() + x.shape[1] * 2.0 ** -44 + 2.0 ** -39
    live = torch.isfinite(wlogp)
    assert torch.equal(torch.isfinite(logp), live)
    assert bool(((logp - wlogp).abs()[live] <= tol[live]).all())
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,V", [(1, 1), (3, 7), (40, 300), (17, 2048), (5, 50001), (3, 152064)])
def test_kernel(B, V, kind, dtype):
    on_gpu(logits_of(kind, B, V, seed=V, dtype=dtype), *settings(B, seed=V + B))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", ["k", "p", "m", "kp", ""])
def test_each_filter_alone_on_a_decode_batch(which, dtype):
    B = 40
    x = logits_of("tail", B, 152064, seed=1, dtype=dtype)
    g = torch.Generator().manual_seed(2)
    u = torch.rand(B, generator=g, dtype=torch.float64)
    on_gpu(x, u, torch.full((B,), 0.8), torch.full((B,), 50, dtype=torch.int32) if "k" in which else None,
           torch.full((B,), 0.9) if "p" in which else None, torch.full((B,), 0.05) if "m" in which else None)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [512, 4099, 152064])
def test_large_k_and_flat_rows(V):
    B = 6
    x = logits_of("normal", B, V, seed=3, dtype=torch.bfloat16) * 0.1
    u = torch.rand(B, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    for k in (V // 2, V - 1, V, 3 * V):
        on_gpu(x, u, None, torch.full((B,), k, dtype=torch.int32), torch.full((B,), 0.97))


@pytest.mark.gpu
def test_ends_of_u():
    x = logits_of("coarse", 8, 3000, seed=5)
    u = torch.tensor([0.0, 2.0 ** -60, 1 - 2.0 ** -53, 0.5] * 2, dtype=torch.float64)
    on_gpu(x, u)
    on_gpu(x, u, None, torch.full((8,), 7, dtype=torch.int32))
    # past the ends: the first and the last kept token
    a = ops.sample(x.cuda(), torch.full((8,), -1.0, dtype=torch.float64, device="cuda"))
    b = ops.sample(x.cuda(), torch.full((8,), 1.5, dtype=torch.float64, device="cuda"))
    assert torch.equal(a, on_gpu(x, torch.zeros(8, dtype=torch.float64)))
    assert torch.equal(b, on_gpu(x, torch.full((8,), 1 - 2.0 ** -53, dtype=torch.float64)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e-30, 1e-4, 50.0, 1e30, INF, float("nan"), -1.0])
def test_temperatures(T):
    x = logits_of("tail", 9, 5000, seed=6, dtype=torch.bfloat16)
    u = torch.rand(9, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
    on_gpu(x, u, torch.full((9,), T), None, torch.full((9,), 0.9))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_row_strides_and_odd_starts(dtype):
    base = logits_of("tail", 6, 3011, seed=8, dtype=dtype).cuda()
    s = settings(6, seed=9)
    for lo, hi in ((0, 3011), (1, 3000), (3, 2998), (5, 6), (7, 3011)):
        on_gpu(base[:, lo:hi], *s)
    on_gpu(base[::2, 2:], *(v[:3] for v in s))
    on_gpu(base[1:2].expand(6, 3011), *s)


@pytest.mark.gpu
def test_a_row_does_not_depend_on_its_batch():
    """The same row alone, among 16 and among 200 (other cluster sizes)."""
    x = logits_of("tail", 200, 20000, seed=10, dtype=torch.bfloat16).cuda()
    s = [v.cuda() for v in settings(200, seed=11)]
    full, flp = ops.sample(x, *s, return_logprobs=True)
    for n in (1, 16):
        ids, lp = ops.sample(x[:n], *(v[:n].contiguous() for v in s), return_logprobs=True)
        assert torch.equal(ids, full[:n]) and torch.equal(lp, flp[:n])


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    x = logits_of("tail", 12, 9000, seed=12, dtype=torch.bfloat16).cuda()
    s = [v.cuda() for v in settings(12, seed=13)]
    out = torch.empty(12, dtype=torch.int32, device="cuda")
    ops.sample(x, *s, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, *s, out=out)
    for seed in (14, 15):
        x.copy_(logits_of("tail", 12, 9000, seed=seed, dtype=torch.bfloat16))
        for v, n in zip(s, settings(12, seed=seed)):
            v.copy_(n)
        graph.replay()
        assert torch.equal(out, ref.sample(x, *s)[0])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        y = ops.sample(x, *s)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(y, out)


@pytest.mark.gpu
def test_largest_vocabulary():
    x = torch.zeros(1, 1 << 19, dtype=torch.bfloat16, device="cuda")
    for u in (0.0, 0.25, 1 - 2.0 ** -30):
        assert int(ops.sample(x, torch.tensor([u], dtype=torch.float64, device="cuda"))) == int(u * 2 ** 19)


@pytest.mark.gpu
@pytest.mark.parametrize("V,dtype", [(1 << 19, torch.bfloat16), (389000, torch.float32)])
def test_longest_rows(V, dtype):
    on_gpu(logits_of("tail", 3, V, seed=12, dtype=dtype), *settings(3, seed=13))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1023, 1024, 1025, 2049])
@pytest.mark.parametrize("k", [1, 2, 127, 128, 129, 1000, 1024, 1025])
def test_numbers_of_candidates_at_which_the_way_changes(k, V):
    """One warp, one CTA, the whole cluster; the row listed whole or not."""
    B = 12
    x = logits_of("coarse", B, V, seed=k, dtype=torch.bfloat16)
    u = torch.rand(B, generator=torch.Generator().manual_seed(k + V), dtype=torch.float64)
    kk = torch.full((B,), k, dtype=torch.int32)
    p = torch.linspace(0.05, 1.0, B)
    on_gpu(x, u, None, kk)
    on_gpu(x, u, None, kk, p)
    on_gpu(x, u, None, None, p)
    on_gpu(x, u, None, kk, p, torch.full((B,), 1e-3))


@pytest.mark.gpu
def test_refusals():
    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    ops.sample(x, u)
    for bad in (dict(logits=x.half()), dict(logits=x.t()), dict(logits=torch.zeros(2, (1 << 19) + 1, device="cuda")),
                dict(logits=torch.zeros(2, 0, device="cuda")), dict(logits=torch.zeros(1, 1 << 19, device="cuda"), uniforms=u[:1]),
                dict(uniforms=u.float()), dict(uniforms=u[:1]), dict(uniforms=u.cpu()), dict(temperature=u),
                dict(top_k=torch.zeros(2, device="cuda")), dict(top_p=torch.ones(3, device="cuda")),
                dict(min_p=torch.ones(4, device="cuda")[::2]), dict(out=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            ops.sample(**{"logits": x, "uniforms": u, **bad})
    assert ops.sample(x[:0], u[:0]).shape == (0,)
