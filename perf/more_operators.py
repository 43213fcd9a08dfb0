"""What the operators of the projections in 8 bits are measured on.

A matrix in 8 bits is e4m3 values with one fp32 scale a row,

    s[m] = max(max_k |y[m, k]| / 448, 2^-126),   q[m, k] = e4m3(y[m, k] / s[m]),

448 being the largest e4m3 number; a row with an infinity or a NaN has the
scale NaN.

``quantize_q8``: y = x.
``rmsnorm_q8``, ``fused_add_rmsnorm_q8``: y = x rsqrt(mean x^2 + eps) w; the
latter with x + residual in the place of x, which is stored as well.
``linear_q8``: a projection whose input and weight are in 8 bits,

    y[m, n] = s[m] t[n] sum_k q[m, k] p[n, k] + bias[n],

optionally followed by silu(gate) * up of an interleaved gate/up product, and
by the addition of a residual.
"""

import math

import torch

own = False

EPS = 1e-6


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one agent decoding: the first norm of a layer of Qwen2.5-7B
        dict(name="norm_1", op="norm", M=1, K=3584, add=False),
        # a decode batch of 16 on Qwen3-32B: the residual's addition with the norm
        dict(name="norm_add_16", op="norm", M=16, K=5120, add=True),
        # the repair rows of a 16K Link on Qwen2.5-7B
        dict(name="norm_add_5087", op="norm", M=5087, K=3584, add=True),
        # a short prompt on the small test model: a matrix whose rows are part of wider ones
        dict(name="quantize_300_small", op="quantize", M=300, K=512, pad=64),
        # the gated rows of a 2048-row prefill, ahead of the down projection
        dict(name="quantize_2048_wide", op="quantize", M=2048, K=18944, pad=0),
        # one agent decoding: the qkv projection of Qwen2.5-7B
        dict(name="linear_decode_1", op="linear", M=1, K=3584, N=4608, bias=True, residual=False, swiglu=False),
        # a decode batch of 16: the gate/up projection with its SwiGLU
        dict(name="linear_decode_16_swiglu", op="linear", M=16, K=3584, N=37888, bias=False, residual=False, swiglu=True),
        # an odd decode batch: the o projection of Qwen3-32B, added to the residual
        dict(name="linear_decode_61", op="linear", M=61, K=8192, N=5120, bias=False, residual=True, swiglu=False),
        # a short prompt on the small test model
        dict(name="linear_prompt_300_small", op="linear", M=300, K=512, N=1024, bias=True, residual=False, swiglu=False),
        # the repair rows of a 16K Link: the qkv projection
        dict(name="linear_prompt_5087", op="linear", M=5087, K=3584, N=4608, bias=True, residual=False, swiglu=False),
        # a 2048-row prefill batch: the gate/up projection with its SwiGLU
        dict(name="linear_prompt_2048_swiglu", op="linear", M=2048, K=3584, N=37888, bias=False, residual=False, swiglu=True),
        # the repair rows again: the down projection, added to the residual
        dict(name="linear_prompt_5087_down", op="linear", M=5087, K=18944, N=3584, bias=False, residual=True, swiglu=False),
    ]


MOST = 5087 * 18944 * 3584


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.random()
    if kind < 0.25:
        return dict(op="norm", M=_log_int(rng, 1, 8000), K=16 * _log_int(rng, 4, 768), add=rng.random() < 0.5)
    if kind < 0.4:
        return dict(op="quantize", M=_log_int(rng, 1, 5000), K=16 * _log_int(rng, 4, 1600), pad=rng.choice([0, 0, 8, 64]))
    M = _log_int(rng, 1, 5000)
    K = 16 * _log_int(rng, 4, 1600)
    swiglu = rng.random() < 0.4
    N = 32 * _log_int(rng, 4, 1184) if swiglu else 8 * _log_int(rng, 16, 4736)
    while M * N * K > MOST:
        M = (M + 1) // 2
    return dict(op="linear", M=M, K=K, N=N, bias=rng.random() < 0.5, residual=rng.random() < 0.5, swiglu=swiglu)


# ------------------------------------------------------------------ inputs
def _rows_q8(y):
    """A program's matrix in 8 bits, kept from before the call."""
    scale = (y.abs().amax(dim=1, keepdim=True) / 448.0).clamp(min=2.0 ** -126)
    return (y / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale[:, 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    M, K = case["M"], case["K"]
    if case["op"] == "linear":
        N = case["N"]
        st = {"case": case, "bias": normal(N).mul_(0.1).to(torch.bfloat16) if case["bias"] else None}
        # rows of different sizes, a few large channels
        st["x"] = _rows_q8(normal(M, K) * torch.exp(0.5 * normal(M, 1)) * torch.exp(0.3 * normal(K)))
        st["w"] = _rows_q8(normal(N, K) * 0.02)
        out = N // 2 if case["swiglu"] else N
        st["residual"] = normal(M, out).to(torch.bfloat16) if case["residual"] else None
        return st
    if case["op"] == "quantize":
        wide = (normal(M, K + case["pad"]) * torch.exp(normal(M, 1))).to(torch.bfloat16)
        return {"case": case, "x": wide[:, :K]}
    # a residual stream: some channels carry much larger values than the others
    channel = torch.exp(0.5 * normal(K)) * torch.where(torch.rand(K, generator=g, device="cuda") < 0.002, 30.0, 1.0)
    st = {"case": case, "x": (normal(M, K) * channel).to(torch.bfloat16), "w": (1.0 + 0.1 * normal(K)).to(torch.bfloat16)}
    if case["add"]:
        st["residual"] = (2.0 * normal(M, K) * channel).to(torch.bfloat16)
        st["sum"] = torch.empty_like(st["residual"])
    return st


# -------------------------------------------------------------- plain forms
def _plain_q8(y):
    top = y.abs().amax(dim=1, keepdim=True)
    scale = torch.clamp(top / 448.0, min=2.0 ** -126)
    scale = torch.where(top < math.inf, scale, torch.full_like(scale, math.nan))
    return (y * (1.0 / scale)).to(torch.float8_e4m3fn), scale[:, 0]


def _plain_norm(st):
    y = st["x"].float()
    if st["case"]["add"]:
        y = y + st["residual"].float()
        st["sum"].copy_(y)
    rstd = torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS)
    q, scale = _plain_q8(y * rstd * st["w"].float())
    return (q, scale, st["sum"]) if st["case"]["add"] else (q, scale)


def _plain_linear(st):
    (xq, xs), (wq, ws) = st["x"], st["w"]
    y = (xq.float() @ wq.float().t()) * xs[:, None] * ws
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["case"]["swiglu"]:
        M, N = y.shape
        y = y.view(M, N // 32, 2, 16)
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(M, N // 2)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(torch.bfloat16)


def run(state):
    case = state["case"]
    if own:
        from sglang_legolink_b200 import ops

        if case["op"] == "linear":
            return ops.linear_q8(ops.Q8(*state["x"]), ops.Q8(*state["w"]), state["bias"], residual=state["residual"],
                                 swiglu_epilogue=case["swiglu"])
        if case["op"] == "quantize":
            return tuple(ops.quantize_q8(state["x"]))
        if not case["add"]:
            return tuple(ops.rmsnorm_q8(state["x"], state["w"], EPS))
        q = ops.fused_add_rmsnorm_q8(state["x"], state["residual"], state["w"], EPS, residual_out=state["sum"])
        return q.values, q.scale, state["sum"]
    if case["op"] == "linear":
        return _plain_linear(state)
    return _plain_q8(state["x"].float()) if case["op"] == "quantize" else _plain_norm(state)


# -------------------------------------------------------------------- work
def work(case):
    M, K = case["M"], case["K"]
    if case["op"] == "linear":
        N = case["N"]
        out = N // 2 if case["swiglu"] else N
        moved = M * K + N * K + 4 * (M + N) + 2 * M * out + (2 * N if case["bias"] else 0)
        return {"bytes": moved + (2 * M * out if case["residual"] else 0), "flops": 2 * M * N * K}
    if case["op"] == "quantize":
        # a magnitude, a maximum and a product for each value
        return {"bytes": 3 * M * K + 4 * M, "flops": 3 * M * K}
    # besides, a square, a sum and two products, and the addition
    return {"bytes": M * K * (7 if case["add"] else 3) + 2 * K + 4 * M, "flops": M * K * (8 if case["add"] else 7)}


# ------------------------------------------------------------ in 64 bits
def _exact_q8(y):
    top, _ = torch.max(torch.abs(y), dim=1)
    scale = torch.maximum(top / 448, torch.full_like(top, 2.0 ** -126))
    v = y / scale[:, None]
    # numbers of three bits behind the point, their exponent at least -6
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(torch.abs(v), min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step, scale


def _exact_linear(st):
    x, w = (q.to(torch.float64) * s.to(torch.float64).unsqueeze(1) for q, s in (st["x"], st["w"]))
    y = torch.matmul(x, torch.transpose(w, 0, 1))
    if st["bias"] is not None:
        y += st["bias"].to(torch.float64)
    if st["case"]["swiglu"]:
        cols = torch.arange(y.shape[1], device=y.device)
        gate, up = y[:, cols % 32 < 16], y[:, cols % 32 >= 16]
        y = gate * torch.sigmoid(gate) * up
    return y if st["residual"] is None else y + st["residual"].to(torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(st)
    y = st["x"].to(torch.float64)
    if case["op"] == "quantize":
        return _exact_q8(y)
    if case["add"]:
        y = y + st["residual"].to(torch.float64)
    norm = torch.sqrt(torch.sum(torch.square(y), dim=1) / case["K"] + EPS)
    q, scale = _exact_q8(y / norm.unsqueeze(1) * st["w"].to(torch.float64))
    return (q, scale, y) if case["add"] else (q, scale)
