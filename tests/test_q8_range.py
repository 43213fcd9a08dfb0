"""The product of two matrices in 8 bits (``ops.linear_q8``) over the whole range
of its operands and sizes.

Tolerances.  The kernels add 32 products at a time to a sum in fp32, and then the
partial sums of at most eight CTAs: K / 32 + 8 steps.  A step is off by at most
2^-22 of the larger of the sum so far and its products, however it rounds; with
terms of random signs that is at most 6 sqrt(sum of the terms' squares), so a
product is off by (K / 32 + 8) 2^-22 of that, and by six steps of 2^-24 of
itself for the scales, the bias and the residual.  silu(g) u is off by what g and u
are off by (|silu'| <= 1.1) and, relatively, by the fast exponential's 2^-21 and 2^-23
of its argument, as long as exp(-g) is within fp32, |g| < 90; where 1 + exp(-g) is past
2^126 silu(g) is 0, which is off by less than 2^-119.  The result is rounded once,
2^-8 of itself; below bf16's normal numbers, a step is 2^-133.
"""

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.ops import Q8
from test_q8_ops import KERNELS, check_rows_q8, integers_q8, norm64, q8_like, raw, rows_like

gpu = pytest.mark.gpu


def result64(x, w, bias, residual, swiglu):
    """The result in 64 bits and how far one may be off."""
    a, b = (t.values.cpu().double() * t.scale.cpu().double()[:, None] for t in (x, w))
    y = a @ b.t()
    tol = (a.shape[1] / 32 + 8) * 2.0 ** -22 * 6 * torch.sqrt((a * a) @ (b * b).t()) + 2.0 ** -22 * y.abs()
    if bias is not None:
        y = y + bias.cpu().double()
        tol = tol + 2.0 ** -23 * y.abs()
    if swiglu:
        c = torch.arange(y.shape[1])
        g, u, tg, tu = y[:, c % 32 < 16], y[:, c % 32 >= 16], tol[:, c % 32 < 16], tol[:, c % 32 >= 16]
        s = g * torch.sigmoid(g)
        y = s * u
        tol = 1.1 * tg * (u.abs() + tu) + s.abs() * tu + (2.0 ** -20 + 2.0 ** -22 * g.abs().clamp(max=90)) * y.abs()
        tol = tol + 2.0 ** -119 * u.abs()
    if residual is not None:
        y = y + residual.cpu().double()
        tol = tol + 2.0 ** -23 * y.abs()
    return y, tol * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs() + 2.0 ** -133


def far_rows(M, K, N, swiglu, device="cpu"):
    """Rows of x of very different sizes, up to 1e37, against weights of ordinary
    size: results within bf16's range whose factors may leave fp32's.  With SwiGLU
    the up rows are 1e-34 as large, so that gate times up stays finite."""
    g = torch.Generator().manual_seed(11)
    size = torch.tensor([1e36, 1.0, 1e35, 1e-30, 3e37 if not swiglu else 1e34, 1e20])[torch.arange(M) % 6]
    x, w = q8_like(M, K, 12), q8_like(N, K, 13)
    x = Q8(x.values, (size / 448 * (0.5 + torch.rand(M, generator=g))).float())
    ws = 0.05 / 448 * (0.5 + torch.rand(N, generator=g))
    if swiglu:
        ws = torch.where(torch.arange(N) % 32 < 16, ws, ws * 1e-34)
    w = Q8(w.values, ws.float())
    bias = rows_like(1, N, 14)[0].contiguous() * 1e-30
    residual = rows_like(M, N // 2 if swiglu else N, 15) * 1e30
    return tuple(Q8(*(t.to(device) for t in q)) for q in (x, w)) + (bias.to(device), residual.to(device))


@pytest.mark.parametrize("swiglu", [False, True])
def test_rows_of_large_numbers(swiglu):
    """The bf16 product of such rows is finite, and so is this one."""
    x, w, b, r = far_rows(13, 512, 96, swiglu)
    want, tol = result64(x, w, b, r, swiglu)
    assert 1e36 < float(want.abs().max()) < 2e38
    y = ops.linear_q8(x, w, b, residual=r, swiglu_epilogue=swiglu)
    assert torch.all((y.double() - want).abs() <= tol)


@gpu
@pytest.mark.parametrize("kernel", [0] + KERNELS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M", [1, 16, 61, 300])
def test_rows_of_large_numbers_on_the_gpu(M, swiglu, kernel):
    x, w, b, r = far_rows(M, 512, 160, swiglu, "cuda")
    for bias, res in ((None, None), (b, r)):
        want, tol = result64(x, w, bias, res, swiglu)
        y = raw(x, w, bias, res, swiglu, kernel)
        assert torch.all((y.cpu().double() - want).abs() <= tol)


@gpu
@pytest.mark.parametrize("K,N", [(64, 64), (16, 128), (128, 8)])
def test_more_row_tiles_than_a_grid_has_places(K, N):
    """65535 tiles of 128 rows and one row more, of few and short features."""
    M = 65535 * 128 + 1
    x = Q8(torch.randint(-3, 4, (M, K), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda",
                         dtype=torch.int8).to(torch.float8_e4m3fn), torch.full((M,), 0.5, device="cuda"))
    w = integers_q8(N, K, 2, "cuda")
    y = ops.linear_q8(x, w)
    for rows in (slice(0, 300), slice(M // 2, M // 2 + 300), slice(M - 300, M)):
        want = x.values[rows].double() @ w.values.double().t() * 0.5 * w.scale.double()
        assert torch.equal(y[rows], want.to(torch.bfloat16))
    assert bool(torch.isfinite(y).all()) and ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 128, 128), (16, 3584, 512), (61, 8192, 640), (128, 18944, 256), (300, 2048, 1056)])
def test_a_call_that_gives_up_stores_whole_results_only(M, K, N, swiglu, kernel):
    """With an error on record waits return at once: what a call stores all the
    same is right, and the rest of its output is left as it was."""
    gives_up(integers_q8(M, K, 1, "cuda"), integers_q8(N, K, 2, "cuda"), swiglu, kernel)


@gpu
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("swiglu", [False, True])
def test_a_long_call_that_gives_up_leaves_its_output(swiglu, kernel):
    """A product that takes longer than the waits for it look away from the error word."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = (Q8(torch.randint(-3, 4, (R, 1 << 22), generator=g, device="cuda", dtype=torch.int8).to(torch.float8_e4m3fn),
               torch.ones(R, device="cuda")) for R in (16, 64))
    gives_up(x, w, swiglu, kernel)


def gives_up(x, w, swiglu, kernel):
    M, N = x.values.shape[0], w.values.shape[0]
    r = torch.randint(-64, 65, (M, N // 2 if swiglu else N)).to(torch.bfloat16).cuda()
    err = ops.workspace("cuda").err
    for res in (None, r):
        want = raw(x, w, None, res, swiglu, kernel)
        for _ in range(5):
            out = torch.full_like(want, 1234.0)
            err.fill_(6)
            ops._cuda().q8_linear(x.values, x.scale, w.values, w.scale, None, res, out, swiglu, kernel, err)
            assert ops.check_errors("cuda") == 6
            assert bool(((out == want) | (out == 1234)).all())
        assert torch.equal(raw(x, w, None, res, swiglu, kernel), want)
    assert ops.check_errors("cuda") == 0


# ------------------------------------------------- every cluster, long sums
CLUSTERS = [4, 5, 6, 7, 12, 14, 15, 16, 17]  # CTAs to a feature tile that the rules choose beside those of KERNELS


@gpu
@pytest.mark.parametrize("kernel", CLUSTERS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 640, 128), (9, 1808, 160), (29, 512, 96), (33, 1040, 288), (61, 3584, 352), (64, 128, 128),
                                   (125, 1808, 288), (128, 8192, 128), (150, 912, 64)])
def test_clusters_of_every_size(M, K, N, swiglu, kernel):
    """Groups of rows and k-blocks that do not divide among the CTAs; some CTAs have none."""
    x, w = integers_q8(M, K, 1, "cuda"), integers_q8(N, K, 2, "cuda")
    b = torch.randint(-64, 65, (N,), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    cols = N // 2 if swiglu else N
    r = torch.randint(-64, 65, (M, cols), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    for bias, res in ((None, None), (b, r)):
        y = raw(x, w, bias, res, swiglu, kernel).cpu().double()
        want, tol = result64(x, w, bias, res, swiglu)
        # without SwiGLU every step is exact, and the result is rounded once
        ok = (y - want).abs() <= tol if swiglu else y == want.to(torch.bfloat16).double()
        assert torch.all(ok)
    assert ops.check_errors("cuda") == 0


def wide_whole(M, N, K, device="cpu"):
    """Whole numbers whose running sum rises to 2^21 or 2^22 over the first half of K and
    falls back over the second, with small ones beside them: each sum of any part
    is a whole number below 2^24, exact in fp32, and the end is what the small ones give."""
    g = torch.Generator().manual_seed(K)
    big = 2.0 ** (6 if K <= 8192 else 5)
    x, w = (torch.randint(-3, 4, (R, K), generator=g).float() for R in (M, N))
    k = torch.arange(K)
    x[:, k % 4 == 0] = big
    w[:, (k % 4 == 0) & (k < K // 2)] = big
    w[:, (k % 4 == 0) & (k >= K // 2)] = -big
    scale = [torch.exp2(torch.randint(-3, 4, (R,), generator=g).float()) for R in (M, N)]
    return tuple(Q8(t.to(torch.float8_e4m3fn).to(device), s.to(device)) for t, s in zip((x, w), scale))


def product_of(x, w, ks=slice(None)):
    a, b = (t.values.cpu().double()[:, ks] for t in (x, w))
    return a @ b.t() * x.scale.cpu().double()[:, None] * w.scale.cpu().double()


@pytest.mark.parametrize("K", [8192, 18944])
def test_the_long_sums_tell_mistakes_apart(K):
    """Of products without an MMA's 32 values, or whose sum keeps 14 bits, few pass."""
    x, w = wide_whole(61, 128, K)
    want = product_of(x, w).to(torch.bfloat16)
    assert float((want.double() / x.scale[:, None] / w.scale).abs().max()) < 2 ** 12
    for at in (0, 32 * (K // 64), K - 32):
        keep = torch.ones(K, dtype=torch.bool)
        keep[at:at + 32] = False
        assert float((product_of(x, w, keep).to(torch.bfloat16) == want).float().mean()) < 0.2
    total = torch.zeros(61, 128, dtype=torch.float64)
    for k in range(0, K, 32):
        total += x.values.double()[:, k:k + 32] @ w.values.double()[:, k:k + 32].t()
        step = torch.exp2(torch.floor(torch.log2(total.abs().clamp(min=1))) - 13)
        total = torch.trunc(total / step) * step
    cut = (total * x.scale.double()[:, None] * w.scale.double()).to(torch.bfloat16)
    assert float((cut == want).float().mean()) < 0.2


@gpu
@pytest.mark.parametrize("kernel", KERNELS + CLUSTERS)
@pytest.mark.parametrize("M", [1, 61, 128, 300])
@pytest.mark.parametrize("K", [8192, 18944])
def test_long_sums_are_exact(K, M, kernel):
    N = 264
    x, w = wide_whole(M, N, K, "cuda")
    want = product_of(x, w)
    assert torch.equal(raw(x, w, kernel=kernel).cpu(), want.to(torch.bfloat16))
    b = torch.randint(-64, 65, (N,), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    r = torch.randint(-64, 65, (M, N), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    y = raw(x, w, b, r, kernel=kernel)
    assert torch.equal(y.cpu(), (want + b.cpu().double() + r.cpu().double()).to(torch.bfloat16))
    assert ops.check_errors("cuda") == 0


LONG = [(5, 18944, 96), (61, 8192, 640), (128, 18944, 160), (300, 8192, 288)]


@pytest.mark.parametrize("M,K,N", LONG[:2])
def test_the_bound_of_a_long_product_is_sharp(M, K, N):
    """A product without an MMA's 32 values is refused nearly everywhere."""
    x, w = q8_like(M, K, 1), q8_like(N, K, 2)
    want, tol = result64(x, w, None, None, False)
    for at in (0, 32 * (K // 64), K - 32):
        keep = torch.ones(K, dtype=torch.bool)
        keep[at:at + 32] = False
        off = (product_of(x, w, keep).to(torch.bfloat16).double() - want).abs() > tol
        assert float(off.float().mean()) > 0.7


@gpu
@pytest.mark.parametrize("kernel", KERNELS + CLUSTERS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,K,N", LONG)
def test_long_products(M, K, N, swiglu, kernel):
    x, w = q8_like(M, K, 1, "cuda"), q8_like(N, K, 2, "cuda")
    w = Q8(w.values, w.scale * 0.02)
    b = rows_like(1, N, 3, device="cuda")[0].contiguous()
    r = rows_like(M, N // 2 if swiglu else N, 4, 8, "cuda")
    for bias, res in ((None, None), (b, r)):
        want, tol = result64(x, w, bias, res, swiglu)
        assert torch.all((raw(x, w, bias, res, swiglu, kernel).cpu().double() - want).abs() <= tol)


@gpu
@pytest.mark.parametrize("M", [1, 40, 100, 300])
@pytest.mark.parametrize("swiglu", [False, True])
def test_what_lies_beside_the_output_stays(M, swiglu):
    """Rows and columns of a larger buffer, with a width that ends inside the kernels' boxes."""
    K, N = 272, 544 if swiglu else 520
    cols = N // 2 if swiglu else N
    x, w = integers_q8(M, K, 1, "cuda"), integers_q8(N, K, 2, "cuda")
    want = ops.linear_q8(x, w, swiglu_epilogue=swiglu)
    for kernel in [0] + KERNELS:
        buf = torch.full((M + 3, cols + 40), 7.0, dtype=torch.bfloat16, device="cuda")
        out = buf[1:M + 1, 16:cols + 16]
        ops._cuda().q8_linear(x.values, x.scale, w.values, w.scale, None, None, out, swiglu, kernel, ops.workspace("cuda").err)
        if not swiglu:
            assert torch.equal(out, want)
        buf[1:M + 1, 16:cols + 16] = 7
        assert bool((buf == 7).all())


@gpu
@pytest.mark.parametrize("M", [1, 40, 70])
def test_more_feature_tiles_than_a_grid_has_places(M):
    K, N = 16, 65535 * 128 + 8
    x = integers_q8(M, K, 1, "cuda")
    w = Q8(torch.randint(-3, 4, (N, K), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda",
                         dtype=torch.int8).to(torch.float8_e4m3fn), torch.full((N,), 0.5, device="cuda"))
    y = ops.linear_q8(x, w)
    for cols in (slice(0, 300), slice(N // 2, N // 2 + 300), slice(N - 300, N)):
        want = x.values.double() @ w.values[cols].double().t() * 0.5 * x.scale[:, None].double()
        assert torch.equal(y[:, cols], want.to(torch.bfloat16))
    assert bool(torch.isfinite(y).all()) and ops.check_errors("cuda") == 0


def small_rows(K):
    """Rows whose squares leave fp32 at its lower end, down to bf16's least number."""
    x = torch.randn(7, K, generator=torch.Generator().manual_seed(3))
    return (x * torch.tensor([1.0, 1e-12, 1e-18, 1e-20, 1e-25, 1e-36, 0.0])[:, None]).to(torch.bfloat16).index_fill_(
        0, torch.tensor([6]), 2.0 ** -133)


@pytest.mark.parametrize("K", [64, 4096])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-30])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_norm_of_small_rows_with_a_small_eps(K, eps, device):
    x, r = small_rows(K).to(device), (small_rows(K).flip(1) / 2).to(device)
    w = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).to(device)
    check_rows_q8(ops.rmsnorm_q8(x, w, eps), norm64(x, w, eps)[0], 2e-5)
    want, s = norm64(x, w, eps, r)
    check_rows_q8(ops.fused_add_rmsnorm_q8(x, r, w, eps), want, 2e-5)
    assert torch.equal(r.cpu(), s.to(torch.bfloat16))
    none = ops.rmsnorm_q8(torch.zeros(2, K, dtype=torch.bfloat16, device=device), w, eps)
    assert bool(none.scale.isnan().all()) if eps == 0 else bool((none.values.float() == 0).all())
