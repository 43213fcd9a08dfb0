"""Matrices in 8 bits (``ops.quantize_q8``, ``ops.rmsnorm_q8``,
``ops.fused_add_rmsnorm_q8``, ``ops.linear_q8``) against plain statements in 64
bits.

Tolerances.  A value in 8 bits is off by half an e4m3 step: 2^-4 of itself, or
2^-10 of the scale where it is below e4m3's normal numbers.  A norm's fp32 steps
(at most 64 squares a thread, then a tree; rsqrt and two products) are below
2e-5 of the value, by which the value may also round apart.  A product's sum has
K fp32 steps of at most 2^-23 of the sum of magnitudes; its result is rounded
to bf16 once, 2^-8 of itself.
"""

import math

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.ops import Q8
from sglang_legolink_b200.ops import reference as ref

E4M3 = torch.float8_e4m3fn
gpu = pytest.mark.gpu


def rows_like(M, K, seed=0, pad=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K + pad, generator=g) * torch.exp(2.0 * torch.randn(M, 1, generator=g))
    return x.to(torch.bfloat16).to(device)[:, :K]


def check_rows_q8(got: Q8, y64: torch.Tensor, slack: float):
    """``got`` stands for ``y64`` to within half an e4m3 step and ``slack`` of the value."""
    q, s = got.values.cpu().double(), got.scale.cpu().double()
    want = (y64.abs().amax(dim=1) / 448).clamp(min=2.0 ** -126)
    assert torch.all((s - want).abs() <= (slack + 2.0 ** -22) * want)
    err = (q * s[:, None] - y64).abs()
    step = torch.maximum(y64.abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10)
    assert torch.all(err <= step * (1 + 2 * slack + 2.0 ** -20) + (slack + 2.0 ** -20) * y64.abs())
    assert torch.all(q.abs() <= 448)


def norm64(x, w, eps, residual=None):
    y = x.cpu().double()
    if residual is not None:
        y = y + residual.cpu().double()
    return y / torch.sqrt((y * y).mean(dim=1, keepdim=True) + eps) * w.cpu().double(), y


def product64(x: Q8, w: Q8, bias, residual, swiglu):
    """The result in 64 bits and the bound of an fp32 sum's error."""
    a, b = (t.values.cpu().double() * t.scale.cpu().double()[:, None] for t in (x, w))
    K = a.shape[1]
    y, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, mag = y + bias.cpu().double(), mag + bias.cpu().double().abs()
    tol = (K + 8) * 2.0 ** -23 * mag
    if swiglu:
        N = y.shape[1]
        c = torch.arange(N)
        g, u, tg, tu = y[:, c % 32 < 16], y[:, c % 32 >= 16], tol[:, c % 32 < 16], tol[:, c % 32 >= 16]
        y = g * torch.sigmoid(g) * u
        # |silu'| <= 1.1; the fast exponential is off by 2^-21 and 2^-23 of its argument
        tol = 1.1 * tg * (u.abs() + tu) + (g * torch.sigmoid(g)).abs() * tu + 2.0 ** -18 * (1 + g.abs()) * y.abs()
    if residual is not None:
        y = y + residual.cpu().double()
        tol = tol + 2.0 ** -23 * y.abs()
    return y, tol + 2.0 ** -8 * y.abs() * (1 + 2.0 ** -7) + tol * 2.0 ** -8


def q8_like(M, K, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    return Q8(*(t.to(device) for t in ref.quantize_q8(y)))


def integers_q8(M, K, seed, device="cpu"):
    """Small whole numbers with powers of two as scales: every sum is exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-3, 4, (M, K), generator=g).float().to(E4M3)
    return Q8(q.to(device), torch.exp2(torch.randint(-3, 4, (M,), generator=g).float()).to(device))


# ------------------------------------------------------------- plain statement
@pytest.mark.parametrize("K", [16, 48, 512, 3584])
def test_statement_stands_for_the_rows(K):
    x = rows_like(9, K)
    check_rows_q8(ops.quantize_q8(x), x.double(), 0.0)
    w = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16)
    check_rows_q8(ops.rmsnorm_q8(x, w, 1e-6), norm64(x, w, 1e-6)[0], 2e-5)
    r = rows_like(9, K, 2)
    want, s = norm64(x, w, 1e-6, r)
    keep = r.clone()
    got = ops.fused_add_rmsnorm_q8(x, r, w, 1e-6, residual_out=(to := torch.empty_like(r)))
    check_rows_q8(got, want, 2e-5)
    assert torch.equal(to, s.to(torch.bfloat16)) and torch.equal(r, keep)
    again = ops.fused_add_rmsnorm_q8(x, r, w, 1e-6)
    assert torch.equal(r, to) and torch.equal(again.values.float(), got.values.float())


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_statement_of_the_product(swiglu, residual, bias):
    M, K, N = 5, 64, 96
    x, w = q8_like(M, K, 0), q8_like(N, K, 1)
    b = rows_like(1, N, 2)[0].contiguous() if bias else None
    r = rows_like(M, N // 2 if swiglu else N, 3) if residual else None
    y = ops.linear_q8(x, w, b, residual=r, swiglu_epilogue=swiglu)
    want, tol = product64(x, w, b, r, swiglu)
    assert y.dtype == torch.bfloat16 and torch.all((y.double() - want).abs() <= tol)
    out = torch.empty(want.shape, dtype=torch.float32)  # another type on the CPU
    assert ops.linear_q8(x, w, b, r, out, swiglu) is out
    assert torch.all((out.double() - want).abs() <= tol)


def special_rows(K):
    """Zeros, one value alone, the least and the largest numbers, values on the borders between two e4m3."""
    big, tiny = 3.3895313892515355e38, 9.183549615799121e-41
    rows = torch.zeros(8, K)
    rows[1, K // 2] = -1.5
    rows[2, :] = tiny
    rows[3, :] = big * torch.where(torch.arange(K) % 3 == 0, -1.0, 0.125)
    rows[4, :] = 448.0 * 2.0 ** -torch.arange(K).float().clamp(max=100)
    rows[5, :] = (16.0 + torch.arange(K) % 17) / 16.0  # 17/16, 19/16, ...: half way
    rows[5, 0] = 448.0
    rows[6, :] = (torch.arange(K) % 9) * 2.0 ** -10    # below the normal numbers, half steps too
    rows[6, 0] = 448.0
    rows[7, :] = 1e-37
    return rows.to(torch.bfloat16)


def test_statement_at_the_ends_of_the_range():
    x = special_rows(64)
    got = ops.quantize_q8(x)
    check_rows_q8(got, x.double(), 0.0)
    assert got.values[0].float().abs().max() == 0 and got.scale[0] == 2.0 ** -126
    assert got.values[1].float().abs().max() == 448
    for bad in (math.inf, -math.inf, math.nan):
        y = x.clone()
        y[1, 3] = bad
        got = ops.quantize_q8(y)
        assert bool(got.scale[1].isnan()) and not bool(got.scale[[0, 2, 3]].isnan().any())
        prod = ops.linear_q8(got, integers_q8(32, 64, 0))
        assert bool(prod[1].isnan().all()) and not bool(prod[4].isnan().any())


# ------------------------------------------------------------------- refusals
def test_refusals():
    x, w = rows_like(4, 64), torch.ones(64, dtype=torch.bfloat16)
    for bad in (rows_like(4, 24), rows_like(4, 8), rows_like(1, 32784), x[0], x[None]):
        with pytest.raises(ValueError):
            ops.quantize_q8(bad)
    with pytest.raises(ValueError):
        ops.rmsnorm_q8(x, w[:48], 1e-6)
    with pytest.raises(ValueError):
        ops.fused_add_rmsnorm_q8(x, x[:3], w, 1e-6)
    with pytest.raises(ValueError):
        ops.fused_add_rmsnorm_q8(x, x.clone(), w, 1e-6, residual_out=x[:, :48])
    with pytest.raises(ValueError):
        ops.quantize_q8(x, out=ops.empty_q8(4, 48, "cpu"))
    with pytest.raises(ValueError):
        ops.quantize_q8(x, out=Q8(torch.empty(4, 64), torch.empty(4)))
    a, b = q8_like(4, 64, 0), q8_like(32, 64, 1)
    for args in ((a, q8_like(32, 48, 1)), (a, q8_like(28, 64, 1)), (a, b, torch.ones(31)), (Q8(a.values.float(), a.scale), b),
                 (Q8(a.values, a.scale[:3]), b), (Q8(a.values, a.scale.double()), b), (Q8(a.values[0], a.scale), b),
                 (a, b, None, torch.ones(4, 31)), (a, b, None, None, torch.ones(3, 32))):
        with pytest.raises(ValueError):
            ops.linear_q8(*args)
    with pytest.raises(ValueError):
        ops.linear_q8(a, q8_like(40, 64, 1), swiglu_epilogue=True)
    with pytest.raises(ValueError):
        ops.linear_q8(a, b, residual=torch.ones(4, 32), swiglu_epilogue=True)


def test_no_rows():
    assert ops.linear_q8(ops.quantize_q8(rows_like(0, 64)), q8_like(32, 64, 1)).shape == (0, 32)


# ----------------------------------------------------------------- on the GPU
ROW_SIZES = [(1, 16), (1, 3584), (3, 48), (7, 256), (8, 272), (9, 1024), (33, 1040), (5, 4096), (2, 4112), (300, 512),
             (4, 8192), (3, 8208), (2, 16384), (3, 18944), (2, 25600), (2, 32768), (700, 3584)]


@gpu
@pytest.mark.parametrize("M,K", ROW_SIZES)
@pytest.mark.parametrize("pad", [0, 24])
def test_quantize_equals_the_statement(M, K, pad):
    """Every step is exactly rounded on both sides: the same bits."""
    x = rows_like(M, K, M, pad)
    want = ops.quantize_q8(x)
    out = ops.empty_q8(M, K, "cuda") if pad else None
    got = ops.quantize_q8(x.cuda() if not pad else rows_like(M, K, M, pad, "cuda"), out=out)
    assert torch.equal(got.scale.cpu(), want.scale)
    assert torch.equal(got.values.cpu().view(torch.uint8), want.values.view(torch.uint8))


@gpu
@pytest.mark.parametrize("K", [64, 2048, 32768])
def test_quantize_at_the_ends_of_the_range(K):
    x = special_rows(K)
    x = torch.cat([x, x[:3]])
    x[8, 1], x[9, K - 1], x[10, K // 2] = math.inf, math.nan, -math.inf
    got, want = ops.quantize_q8(x.cuda()), ops.quantize_q8(x)
    assert torch.equal(got.scale.isnan().cpu(), torch.arange(11) >= 8)
    assert torch.equal(got.scale[:8].cpu(), want.scale[:8])
    assert torch.equal(got.values[:8].cpu().view(torch.uint8), want.values[:8].view(torch.uint8))
    assert bool(got.values[8:].cpu().float().isnan().all())


@gpu
@pytest.mark.parametrize("M,K", ROW_SIZES)
def test_norm(M, K):
    x, r = rows_like(M, K, 1, 8, "cuda"), rows_like(M, K, 2, 16, "cuda")
    w = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).cuda()
    check_rows_q8(ops.rmsnorm_q8(x, w, 1e-6), norm64(x, w, 1e-6)[0], 2e-5)
    want, s = norm64(x, w, 1e-6, r)
    keep, to = r.clone(), torch.full((M, K + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.fused_add_rmsnorm_q8(x, r, w, 1e-6, residual_out=to[:, :K])
    check_rows_q8(got, want, 2e-5)
    assert torch.equal(to[:, :K].cpu(), s.to(torch.bfloat16)) and torch.equal(r, keep)
    assert bool((to[:, K:] == 7).all())
    again = ops.fused_add_rmsnorm_q8(x, r, w, 1e-6)  # in place
    assert torch.equal(r, to[:, :K]) and torch.equal(again.values.view(torch.uint8), got.values.view(torch.uint8))


@gpu
@pytest.mark.parametrize("K", [64, 4096])
def test_norm_of_extreme_rows(K):
    """Squares past fp32's range, rows of zeros, rows far below eps, values that are not finite."""
    x = torch.randn(6, K, generator=torch.Generator().manual_seed(3))
    x[1] *= 1e37
    x[2] = 0
    x[3] *= 1e-38
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    x = x.to(torch.bfloat16)
    w = torch.ones(K, dtype=torch.bfloat16)
    got = ops.rmsnorm_q8(x.cuda(), w.cuda(), 1e-6)
    check_rows_q8(Q8(got.values[:4], got.scale[:4]), norm64(x[:4], w, 1e-6)[0], 2e-5)
    assert bool(got.scale[4:].isnan().all())
    s = ops.rmsnorm_q8(x, w, 1e-6)  # the statement agrees
    check_rows_q8(Q8(s.values[:4], s.scale[:4]), norm64(x[:4], w, 1e-6)[0], 2e-5)
    assert bool(s.scale[4:].isnan().all())


@gpu
@pytest.mark.parametrize("M,K", [(5000, 1040), (2600, 2048), (1400, 3584), (640, 8192)])
def test_many_rows(M, K):
    """More rows than have places at once, some of them extreme: the same bits
    as the statement, and norms as far from 64 bits as those of few rows."""
    x, r = rows_like(M, K, 4), rows_like(M, K, 5)
    x[7], r[7] = 0, 0
    x[8], r[8] = x[8] * 1e30, r[8] * 1e30
    x[9], r[9] = x[9] * 1e-38, r[9] * 1e-38
    x[M - 3, 0], x[M - 2, K // 2], x[M - 1, K - 1] = math.inf, math.nan, -math.inf
    w = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(6))).to(torch.bfloat16)
    ok = slice(0, M - 3)
    got, want = ops.quantize_q8(x.cuda()), ops.quantize_q8(x)
    assert torch.equal(got.scale[ok].cpu(), want.scale[ok]) and bool(got.scale[M - 3:].isnan().all())
    assert torch.equal(got.values[ok].cpu().view(torch.uint8), want.values[ok].view(torch.uint8))
    got = ops.rmsnorm_q8(x.cuda(), w.cuda(), 1e-6)
    check_rows_q8(Q8(got.values[ok], got.scale[ok]), norm64(x[ok], w, 1e-6)[0], 2e-5)
    assert bool(got.scale[M - 3:].isnan().all())
    y, s = norm64(x[ok], w, 1e-6, r[ok])
    total = r.cuda()
    got = ops.fused_add_rmsnorm_q8(x.cuda(), total, w.cuda(), 1e-6)
    check_rows_q8(Q8(got.values[ok], got.scale[ok]), y, 2e-5)
    assert torch.equal(total[ok].cpu(), s.to(torch.bfloat16)) and bool(got.scale[M - 3:].isnan().all())


def raw(x, w, bias=None, residual=None, swiglu=False, kernel=0):
    """The product by a named kernel (64, 128, 256: pairs of CTAs on tiles of so many
    features; up to 8: as many CTAs to a feature tile; 11 to 18: the same, one to a SM)."""
    M, N = x.values.shape[0], w.values.shape[0]
    out = torch.full((M + 2, N // 2 if swiglu else N), 3.0, dtype=torch.bfloat16, device="cuda")
    ops._cuda().q8_linear(x.values, x.scale, w.values, w.scale, bias, residual, out[:M], swiglu, kernel,
                          ops.workspace("cuda").err)
    assert bool((out[M:] == 3).all())
    return out[:M]


KERNELS = [256, 128, 64, 1, 2, 3, 8, 11, 13, 18]


@gpu
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("M,K,N", [(1, 16, 8), (2, 128, 128), (16, 144, 136), (17, 512, 40), (33, 1040, 264), (64, 272, 128),
                                   (65, 384, 520), (129, 640, 256), (255, 128, 248), (257, 3584, 512), (300, 512, 1024),
                                   (513, 1808, 776)])
def test_product_of_whole_numbers_is_exact(M, K, N, kernel):
    x, w = integers_q8(M, K, 1, "cuda"), integers_q8(N, K, 2, "cuda")
    want = (x.values.cpu().double() @ w.values.cpu().double().t()) * x.scale.cpu().double()[:, None] * w.scale.cpu().double()
    y = raw(x, w, kernel=kernel)
    assert torch.equal(y.cpu(), want.to(torch.bfloat16))
    b = torch.randint(-64, 65, (N,)).to(torch.bfloat16).cuda()
    r = torch.randint(-64, 65, (M, N)).to(torch.bfloat16).cuda()
    y = raw(x, w, b, r, kernel=kernel)
    assert torch.equal(y.cpu(), (want + b.cpu().double() + r.cpu().double()).to(torch.bfloat16))
    assert ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 3584, 4608), (5, 18944, 96), (61, 8192, 640), (128, 512, 1024), (300, 1024, 1056),
                                   (700, 2000, 2080)])
def test_product(M, K, N, swiglu, kernel):
    x, w = q8_like(M, K, 1, "cuda"), q8_like(N, K, 2, "cuda")
    w = Q8(w.values, w.scale * 0.02)
    b = rows_like(1, N, 3, device="cuda")[0].contiguous()
    r = rows_like(M, N // 2 if swiglu else N, 4, 8, "cuda")
    for bias, res in ((None, None), (b, r)):
        want, tol = product64(x, w, bias, res, swiglu)
        y = raw(x, w, bias, res, swiglu, kernel)
        assert torch.all((y.cpu().double() - want).abs() <= tol)
        assert torch.equal(y, raw(x, w, bias, res, swiglu, kernel))  # the same bits again
    assert ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("M", [1, 16, 61, 128, 129, 300, 1000])
@pytest.mark.parametrize("swiglu", [False, True])
def test_linear_q8(M, swiglu):
    """The kernel by the rule, rows of wider buffers, the residual in place."""
    K, N = 1040, 1056
    wide = q8_like(M, K + 32, 1, "cuda")
    x, w = Q8(wide.values[:, 16:K + 16], wide.scale), q8_like(N, K, 2, "cuda")
    cols = N // 2 if swiglu else N
    b, r = rows_like(1, N, 3, device="cuda")[0].contiguous(), rows_like(M, cols, 4, 8, "cuda")
    want, tol = product64(x, w, b, r, swiglu)
    y = ops.linear_q8(x, w, b, residual=r, swiglu_epilogue=swiglu)
    assert torch.all((y.cpu().double() - want).abs() <= tol)
    assert ops.linear_q8(x, w, b, residual=r, out=r, swiglu_epilogue=swiglu) is r
    assert torch.equal(r, y)


@gpu
def test_other_rows_do_not_change_a_row():
    x, w = q8_like(100, 512, 1, "cuda"), q8_like(256, 512, 2, "cuda")
    y = ops.linear_q8(x, w)
    other = q8_like(100, 512, 9, "cuda")
    other.values[40], other.scale[40] = x.values[40], x.scale[40]
    other.scale[41] = math.nan
    z = ops.linear_q8(other, w)
    assert torch.equal(z[40], y[40]) and bool(z[41].isnan().all()) and not bool(z[42].isnan().any())


@gpu
def test_a_weight_may_come_from_the_kernel_just_ahead():
    """The product reads nothing before the kernels ahead of it are done."""
    x = integers_q8(16, 2048, 0, "cuda")
    ws = [torch.randint(-3, 4, (1024, 2048), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda()
          for i in range(4)]
    for w in ws:
        w[:, 0] = 448  # the scale is 1
    buf, act = ops.empty_q8(1024, 2048, "cuda"), ops.empty_q8(16, 2048, "cuda")
    want = [(x.values.float() @ w.float().t() * x.scale[:, None]).to(torch.bfloat16) for w in ws]
    rows = (x.values.float() * x.scale[:, None]).to(torch.bfloat16)
    rows[:, 1] = 448.0
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for w in ws:
            ops.quantize_q8(w, out=buf)
            got.append(ops.linear_q8(x, buf))
            ops.quantize_q8(rows, out=act)
        assert all(torch.equal(g, t) for g, t in zip(got, want))


@gpu
def test_captured_and_on_two_streams():
    x, w = rows_like(16, 1024, 1, device="cuda"), ops.quantize_q8(rows_like(512, 1024, 2, device="cuda"))
    g, nw = torch.cuda.CUDAGraph(), torch.ones(1024, dtype=torch.bfloat16, device="cuda")
    r = rows_like(16, 512, 3, device="cuda")

    def step():
        return ops.linear_q8(ops.rmsnorm_q8(x, nw, 1e-6), w, residual=r)

    want = step()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    x.copy_(rows_like(16, 1024, 7, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, step())
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)


@gpu
def test_refusals_on_the_gpu():
    x, w = q8_like(32, 64, 0, "cuda"), q8_like(32, 64, 1, "cuda")
    bf = torch.zeros(32, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):  # fp32 rows
        ops.quantize_q8(bf.float())
    with pytest.raises(RuntimeError):  # rows off the 16-byte boundaries
        ops.quantize_q8(torch.zeros(32, 65, dtype=torch.bfloat16, device="cuda")[:, :64])
    with pytest.raises(RuntimeError):  # the sum where another input is
        ops.fused_add_rmsnorm_q8(bf, bf.clone(), torch.ones(64, dtype=torch.bfloat16, device="cuda"), 1e-6, residual_out=bf)
    with pytest.raises(RuntimeError):  # values over their own input
        ops.quantize_q8(bf, out=Q8(bf.view(E4M3)[:, :64], torch.empty(32, device="cuda")))
    with pytest.raises(RuntimeError):  # another device
        ops.linear_q8(x, Q8(w.values.cpu(), w.scale.cpu()))
    with pytest.raises(RuntimeError):
        ops.linear_q8(x, w, out=torch.zeros(32, 32, device="cuda"))
    with pytest.raises(RuntimeError):  # rows of the output share memory
        ops.linear_q8(x, w, out=torch.zeros(1, 32, dtype=torch.bfloat16, device="cuda").expand(32, 32))
    with pytest.raises(RuntimeError):  # the output over the input
        ops.linear_q8(x, w, out=x.values.view(torch.bfloat16))
    buf = torch.zeros(33, 32, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):  # the output a row behind the residual
        ops.linear_q8(x, w, residual=buf[:32], out=buf[1:])


@gpu
def test_no_rows_on_the_gpu():
    w = q8_like(32, 64, 1, "cuda")
    x = ops.quantize_q8(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"))
    assert x.values.shape == (0, 64) and x.scale.shape == (0,)
    assert ops.linear_q8(x, w).shape == (0, 32)
    r = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert ops.fused_add_rmsnorm_q8(r, r.clone(), torch.ones(64, dtype=torch.bfloat16, device="cuda"), 1e-6).values.numel() == 0


@gpu
def test_offsets_past_32_bits():
    """More than 2^31 values of x and of the result: the last rows are right."""
    M, K = 140000, 16384
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    last = rows_like(3, K, 5, device="cuda")
    x[-3:] = last
    got, want = ops.quantize_q8(x), ops.quantize_q8(last)
    assert torch.equal(got.values[-3:].view(torch.uint8), want.values.view(torch.uint8))
    assert torch.equal(got.scale[-3:], want.scale) and float(got.scale[0]) == 2.0 ** -126
    del x, got
    M, N, K = 70000, 32768, 64
    a, b = integers_q8(M, K, 1, "cuda"), integers_q8(N, K, 2, "cuda")
    r = torch.ones(M, N, dtype=torch.bfloat16, device="cuda")
    y = ops.linear_q8(a, b, residual=r, out=r)
    tail = slice(M - 300, M)
    want = (a.values[tail].double() @ b.values.double().t()) * a.scale[tail, None].double() * b.scale.double() + 1
    assert torch.equal(y[tail], want.to(torch.bfloat16))
    assert ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_row_of_nan_values_stays_its_own(M):
    """NaN codes in one row of x and one of w: that row and that column, whatever lies behind the last row."""
    x, w = q8_like(M, 272, 1, "cuda"), q8_like(136, 272, 2, "cuda")
    want = ops.linear_q8(x, w)
    nan = torch.tensor(math.nan, device="cuda")
    x.values[M // 2] = nan.to(E4M3)
    w.values[7] = nan.to(E4M3)
    y = ops.linear_q8(x, w)
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[M // 2], keep[:, 7] = False, False
    assert torch.equal(y[keep], want[keep]) and bool(y[~keep].isnan().all())


@gpu
def test_two_graphs_replayed_on_two_streams():
    """Nothing but the error word is shared between calls."""
    x, w = q8_like(5, 2048, 1, "cuda"), q8_like(640, 2048, 2, "cuda")
    want = ops.linear_q8(x, w)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(8):
                y = ops.linear_q8(x, w)
        graphs.append(g)
        outs.append(y)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs) and ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("K,N", [(64, 64), (2048, 5120), (18944, 384)])
def test_a_row_alone_and_among_others(K, N):
    """The kernels differ in the order of a row's sums alone."""
    x, w = q8_like(700, K, 1, "cuda"), q8_like(N, K, 2, "cuda")
    want, tol = product64(x, w, None, None, False)
    for M in (1, 16, 17, 33, 64, 65, 128, 129, 256, 257, 700):
        y = ops.linear_q8(Q8(x.values[:M], x.scale[:M]), w)
        assert torch.all((y.cpu().double() - want[:M]).abs() <= tol[:M]), M


@gpu
@pytest.mark.parametrize("kernel", KERNELS)
def test_sums_that_cancel_over_a_wide_range(kernel):
    """Values over the whole of e4m3, the second half of K against the first but
    for a few: the sums of magnitudes are 1e3 to 1e5 times the results."""
    g = torch.Generator().manual_seed(6)

    def wide(R, K):
        v = torch.exp2(torch.randint(-9, 9, (R, K), generator=g).float()) * (1 + torch.randint(0, 8, (R, K), generator=g) / 8)
        return (torch.where(torch.rand(R, K, generator=g) < 0.5, -v, v)).clamp(-448, 448)

    M, K, N = 70, 4096, 264
    x, w = wide(M, K), wide(N, K)
    x[:, K // 2:] = x[:, : K // 2]
    w[:, K // 2:] = -w[:, : K // 2] * torch.where(torch.rand(N, K // 2, generator=g) < 0.01, 0.5, 1.0)
    x, w = (Q8(t.to(E4M3).cuda(), torch.ones(t.shape[0], device="cuda")) for t in (x, w))
    want, tol = product64(x, w, None, None, False)
    assert torch.all((raw(x, w, kernel=kernel).cpu().double() - want).abs() <= tol)


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 256, 256), (40, 512, 384), (300, 128, 512), (1000, 256, 1024)])
def test_results_are_there_for_the_kernel_behind(M, K, N):
    """Every launch may start before the one ahead of it ends: what it reads has to be complete."""
    xs = [q8_like(M, K, s, "cuda") for s in range(4)]
    w, w2 = q8_like(N, K, 9, "cuda"), q8_like(256, N, 10, "cuda")
    norm = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    y, q = torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), ops.empty_q8(M, N, "cuda")
    z, n = torch.empty(M, 256, dtype=torch.bfloat16, device="cuda"), ops.empty_q8(M, 256, "cuda")

    def step(x, wait):
        for f in (lambda: ops.linear_q8(x, w, out=y), lambda: ops.quantize_q8(y, out=q), lambda: ops.linear_q8(q, w2, out=z),
                  lambda: ops.rmsnorm_q8(z, norm, 1e-6, out=n)):
            f()
            if wait:
                torch.cuda.synchronize()
        return n.values.view(torch.uint8).clone(), n.scale.clone()

    want = [step(x, True) for x in xs]
    for _ in range(50):
        got = [step(x, False) for x in xs]
        assert all(torch.equal(a, b) for g, t in zip(got, want) for a, b in zip(g, t))
