"""The projection with per-row low-rank adapters: plan, refusals and the CPU
statement here; the kernels against the formula in 64 bits on a GPU."""

import pytest
import torch

from sglang_legolink_b200 import ops

BF = torch.bfloat16


def make(M, K, N, R, n, rows, seed=0, bias=True, device="cpu", dtype=BF):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)

    if rows == "mixed":
        ids = torch.randint(-1, n, (M,), generator=g)
    elif rows == "runs":
        ids = (torch.arange(M) * 5 // max(1, M)) % (n + 1) - 1
    elif rows == "none":
        ids = torch.full((M,), -1)
    else:
        ids = torch.arange(M) % n
    scale = (0.5 + torch.rand(n, generator=g)).to(device)
    return dict(x=normal(M, K), w=normal(N, K, std=0.05), bias=normal(N, std=0.3) if bias else None,
                a=normal(n, R, K, std=K ** -0.5), b=normal(n, N, R, std=0.2), scale=scale, ids=ids)


def formula64(t, swiglu):
    """The result in float64 and, element by element, how far a kernel may be
    from it: half a bf16 step of the result, half a step of two bf16 terms of
    each low-rank value, and an fp32 rounding per term of each sum."""
    d = lambda v: v.cpu().double()  # noqa: E731
    x, w, a, b, s, ids = d(t["x"]), d(t["w"]), d(t["a"]), d(t["b"]), d(t["scale"]), t["ids"]
    K, R = x.shape[1], a.shape[1]
    y, mag = x @ w.T, x.abs() @ w.abs().T
    if t["bias"] is not None:
        y, mag = y + d(t["bias"]), mag + d(t["bias"]).abs()
    err = torch.zeros_like(y)
    for j in range(a.shape[0]):
        r = (ids == j).nonzero()[:, 0]
        if r.numel():
            low, low_mag = s[j] * (x[r] @ a[j].T), s[j] * (x[r].abs() @ a[j].abs().T)
            y[r] += low @ b[j].T
            term = low.abs() @ b[j].abs().T
            mag[r] += term
            err[r] += 2.0 ** -16 * term + (K + 2) * 2.0 ** -24 * (low_mag @ b[j].abs().T)
    err += (K + R + 2) * 2.0 ** -24 * mag
    if swiglu:
        M, N = y.shape
        v, e = y.view(M, N // 32, 2, 16), err.view(M, N // 32, 2, 16)
        gate, up, eg, eu = (z.reshape(M, N // 2) for z in (v[:, :, 0], v[:, :, 1], e[:, :, 0], e[:, :, 1]))
        silu = gate * torch.sigmoid(gate)
        # |silu'| < 1.1; the fast exponential and the division: within 2^-18
        err = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 2.0 ** -18 * (silu * up).abs()
        y = silu * up
    return y, err + 2.0 ** -8 * (y.abs() + err) + 1e-30


def check(t, swiglu=False, out=None, device="cuda", plan=None):
    dev = torch.device(device)
    stack = ops.LoraStack(t["a"], t["b"], t["scale"])
    plan = plan or ops.lora_plan(t["ids"], dev)
    y = ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan, out=out, swiglu_epilogue=swiglu)
    want, tol = formula64(t, swiglu)
    off = (y.cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the bound"
    if dev.type == "cuda":
        assert ops.check_errors(dev) == 0
    return y


# --------------------------------------------------------------------- CPU
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("M,rows", [(1, "all"), (7, "mixed"), (300, "runs"), (5, "none")])
def test_cpu_statement(M, rows, swiglu):
    t = make(M, 64, 96, 8, 3, rows, seed=M)
    check(t, swiglu, device="cpu")


def test_plan_tiles_planes_and_slots():
    ids = [3, -1, 0, 3, 3, 1]
    p = ops.lora_plan(ids, "cpu")
    assert (p.rows, p.tile_rows, p.tiles, p.max_planes, p.top_adapter) == (6, 128, 1, 3, 3)
    assert p.buf.tolist() == [2, -1, 0, 2, 2, 1] + [0, 3] + [0, 1, 3] + [0, 0, 0]
    ids = [5] * 256 + [2] * 100 + [7] * 156 + [-1] * 10
    p = ops.lora_plan(ids, "cpu")
    assert (p.tile_rows, p.tiles, p.max_planes) == (256, 3, 3)
    assert p.buf[-6:].tolist() == [5, 2, 7, 0, 1, 1] and p.buf[522:526].tolist() == [0, 1, 3, 3]
    assert p.buf[:522].tolist() == [0] * 256 + [0] * 100 + [1] * 156 + [-1] * 10
    assert ops.lora_plan([], "cpu").rows == 0
    assert ops.lora_plan([-1, -1], "cpu").max_planes == 1


def test_plan_update_keeps_the_buffer_and_its_capacity():
    p = ops.lora_plan([0, 1, 2, 0], "cpu", max_planes=3)
    buf = p.buf
    p.update([4, 4, -1, -1])
    assert p.buf is buf and p.top_adapter == 4 and p.buf.tolist() == [0, 0, -1, -1, 0, 1, 4, 0, 0, 0, 0, 0]
    with pytest.raises(ValueError, match="planes"):
        p.update([0, 1, 2, 3])
    with pytest.raises(ValueError, match="rows"):
        p.update([0, 1])
    assert p.buf.tolist() == [0, 0, -1, -1, 0, 1, 4, 0, 0, 0, 0, 0]


def test_stack_pads_different_ranks():
    g = torch.Generator().manual_seed(0)
    pairs = [(torch.randn(r, 32, generator=g), torch.randn(16, r, generator=g)) for r in (4, 12, 1)]
    s = ops.LoraStack.stack(pairs, [1.0, 2.0, 0.5])
    assert s.a.shape == (3, 16, 32) and s.b.shape == (3, 16, 16)
    x = torch.randn(3, 32, generator=g)
    y = ops.linear_lora(x, torch.zeros(16, 32), None, s, ops.lora_plan([0, 1, 2], "cpu"))
    for i, (sc, (a, b)) in enumerate(zip((1.0, 2.0, 0.5), pairs)):
        assert torch.allclose(y[i], sc * (x[i] @ a.T) @ b.T, atol=1e-4)


def test_refusals_on_the_host():
    a, b, s = torch.zeros(2, 8, 32), torch.zeros(2, 16, 8), torch.ones(2)
    for bad in ((a[:, :4], b, s), (a, b[:1], s), (a, b[:, :, :4], s), (a, b, torch.ones(3)),
                (torch.zeros(1, 264, 32), torch.zeros(1, 16, 264), torch.ones(1)), (a, b.double(), s),
                (torch.zeros(0, 8, 32), torch.zeros(0, 16, 8), torch.ones(0))):
        with pytest.raises(ValueError):
            ops.LoraStack(*bad)
    inf = b.clone()
    inf[0, 0, 0] = float("inf")
    with pytest.raises(ValueError, match="finite"):
        ops.LoraStack(a, inf, s)
    stack = ops.LoraStack(a, b, s)
    x, w = torch.zeros(3, 32), torch.zeros(16, 32)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_lora(x, w, None, stack, ops.lora_plan([0, 1], "cpu"))
    with pytest.raises(ValueError, match="adapter"):
        ops.linear_lora(x, w, None, stack, ops.lora_plan([0, 1, 2], "cpu"))
    for bad in ([0.5, 1], [-2, 0], [1 << 31], [[0, 1]]):
        with pytest.raises(ValueError):
            ops.lora_plan(bad, "cpu")


# --------------------------------------------------------------------- GPU
CASES = [  # M, K, N, R, adapters, rows, swiglu
    (1, 512, 1024, 8, 1, "all", False),
    (1, 520, 1000, 24, 3, "all", False),
    (2, 512, 1024, 16, 2, "mixed", True),
    (13, 512, 1024, 48, 13, "all", False),
    (16, 72, 128, 8, 16, "all", False),
    (16, 3584, 4608, 64, 5, "mixed", False),
    (16, 512, 4096, 72, 4, "mixed", True),
    (17, 512, 1024, 256, 3, "mixed", False),
    (33, 1024, 2048, 40, 40, "mixed", True),
    (64, 512, 1024, 16, 64, "all", False),
    (100, 512, 1016, 128, 3, "mixed", False),
    (128, 512, 1024, 16, 128, "all", True),
    (100, 64, 37888, 16, 9, "mixed", False),
    (129, 512, 1024, 8, 2, "runs", False),
    (97, 1024, 512, 256, 3, "mixed", False),  # partials of rows that are no multiple of 32, at large ranks
    (100, 2048, 256, 200, 5, "mixed", True),
    (65, 4096, 128, 256, 40, "all", False),
    (257, 520, 264, 80, 4, "mixed", False),
    (300, 512, 1024, 192, 3, "runs", True),
    (700, 8, 8, 8, 1, "runs", False),
    (1000, 512, 2048, 16, 300, "mixed", False),
    (5, 512, 1024, 16, 2, "none", False),
    (600, 512, 1024, 16, 2, "none", True),
    (255, 1032, 1920, 24, 5, "mixed", False),  # K split past 128 rows
    (513, 264, 1024, 136, 7, "runs", True),
    (1920, 2048, 120, 16, 9, "runs", False),
    (1100, 512, 1920, 16, 6, "runs", False),  # and not: 128 x 128,
    (1100, 520, 1920, 88, 5, "mixed", True),
    (200, 512, 8192, 16, 6, "mixed", False),  # 128 x 256
    (200, 72, 8224, 24, 6, "runs", True),
    (400, 200, 4104, 16, 6, "runs", False),  # and 256 x 256 tiles
    (520, 136, 4096, 104, 6, "mixed", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,n,rows,swiglu", CASES)
def test_against_64_bits(M, K, N, R, n, rows, swiglu):
    check(make(M, K, N, R, n, rows, seed=M + K, device="cuda"), swiglu)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1100, 1920), (200, 8192), (400, 4096)])
def test_a_batch_without_adapters_equals_linear_bit_for_bit(M, N):
    """Where K is not split the tiles and their k-blocks are those of linear()."""
    t = make(M, 512, N, 16, 2, "none", seed=M, device="cuda")
    y = check(t)
    assert torch.equal(y, ops.linear(t["x"], t["w"], t["bias"]))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 300])
def test_strided_rows_and_output(M):
    t = make(M, 512, 1024, 16, 3, "mixed", seed=3, device="cuda")
    wide = torch.randn(M, 640, device="cuda").to(BF)
    wide[:, 64:576] = t["x"]
    t["x"] = wide[:, 64:576]
    buf = torch.full((M + 2, 1152), 7.0, dtype=BF, device="cuda")
    y = check(t, out=buf[1:M + 1, 64:1088])
    assert y.data_ptr() == buf[1:, 64:].data_ptr()
    buf[1:M + 1, 64:1088] = 7.0
    assert bool((buf == 7.0).all()), "the output's neighbours were written"


@pytest.mark.gpu
def test_other_rows_do_not_change_a_row():
    """A row's result does not depend on which adapters the others use."""
    t = make(300, 512, 1024, 16, 8, "mixed", seed=9, device="cuda")
    stack = ops.LoraStack(t["a"], t["b"], t["scale"])
    ids = t["ids"].clone()
    ids[7] = 3
    one = torch.full_like(ids, -1)
    one[7] = 3
    y = ops.linear_lora(t["x"], t["w"], t["bias"], stack, ops.lora_plan(ids, "cuda"))
    z = ops.linear_lora(t["x"], t["w"], t["bias"], stack, ops.lora_plan(one, "cuda"))
    assert torch.equal(y[7], z[7])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [6, 300])
def test_captured_and_replayed_with_other_adapters(M):
    t = make(M, 512, 1024, 16, 6, "mixed", seed=5, device="cuda")
    stack = ops.LoraStack(t["a"], t["b"], t["scale"])
    plan = ops.lora_plan(t["ids"], "cuda", max_planes=12)
    ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan)
    for seed in (1, 2, 3):
        t["ids"] = torch.randint(-1, 6, (M,), generator=torch.Generator().manual_seed(seed))
        plan.update(t["ids"])
        graph.replay()
        want, tol = formula64(t, False)
        assert bool(((y.cpu().double() - want).abs() <= tol).all())
    assert ops.check_errors("cuda") == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["mixed", "none"])
@pytest.mark.parametrize("M,R", [(1, 16), (4, 16), (100, 64), (128, 256), (300, 16), (1100, 16)])
def test_a_chain_of_products_in_a_graph(M, R, rows):
    """Each reads what the one before wrote, with no host between them: a
    kernel that looks at its rows before they are there shows here."""
    H, inter, n = 1024, 2048, 3
    up = make(M, H, 2 * inter, R, n, rows, seed=M, device="cuda")
    down = make(M, inter, H, R, n, rows, seed=M + 1, device="cuda")
    su, sd = (ops.LoraStack(t["a"], t["b"], t["scale"]) for t in (up, down))
    plan = ops.lora_plan(up["ids"], "cuda")

    def chain(wait):
        x, outs = up["x"], []
        for _ in range(4):
            m = ops.linear_lora(x, up["w"], up["bias"], su, plan, swiglu_epilogue=True)
            wait()
            x = ops.linear_lora(m, down["w"], down["bias"], sd, plan)
            x = (x / x.float().norm(dim=1, keepdim=True) * H ** 0.5).to(BF)
            wait()
            outs += [m, x]
        return outs

    want = chain(torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(5):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_two_streams_share_a_stack_and_a_plan():
    t = make(16, 3584, 4608, 16, 5, "mixed", seed=5, device="cuda")
    stack, plan = ops.LoraStack(t["a"], t["b"], t["scale"]), ops.lora_plan(t["ids"], "cuda")
    want = ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.linear_lora(t["x"], t["w"], t["bias"], stack, plan))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    t = make(4, 64, 96, 8, 2, "mixed", device="cuda")
    stack, plan = ops.LoraStack(t["a"], t["b"], t["scale"]), ops.lora_plan([0, 1, -1, 0], "cuda")
    call = lambda x=t["x"], w=t["w"], s=stack, p=plan, **kw: ops.linear_lora(x, w, None, s, p, **kw)  # noqa: E731
    call()
    with pytest.raises(RuntimeError, match="bf16|bfloat16|BFloat16|dtype"):
        call(x=t["x"].float())
    with pytest.raises(RuntimeError):  # K of the projection differs
        call(w=t["w"][:, :56].contiguous())
    with pytest.raises(RuntimeError):  # N of the adapters differs
        call(w=t["w"][:88].contiguous())
    with pytest.raises(RuntimeError):  # rows not on 16-byte boundaries
        call(x=torch.zeros(4, 68, dtype=BF, device="cuda")[:, 4:])
    with pytest.raises(RuntimeError):
        call(out=torch.empty(4, 95, dtype=BF, device="cuda"))
    with pytest.raises(RuntimeError):  # a plan left on the host
        call(p=ops.lora_plan([0, 1, -1, 0], "cpu"))
    assert call(x=t["x"][:0], p=ops.lora_plan([], "cuda")).shape == (0, 96)
