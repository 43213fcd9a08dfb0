"""What the adapter and sampling operators are measured on.

``linear_lora``: a projection shared by every request of a batch, plus each
row's own low-rank adapter,

    y[m] = x[m] W^T + bias + scale[a] (x[m] A[a]^T) B[a]^T,   a = adapter of row m (none: no such term)

optionally followed by silu(gate) * up of an interleaved gate/up product.

``sample``: one token per row of logits from one uniform number per row.
With w_i = exp((x_i - max x) / temperature) and the tokens in descending order
of x (equal ones by index), a row keeps the first ``top_k`` tokens, of those
the ones whose predecessors hold less than ``top_p`` of their mass, and of
those the ones with w_i >= ``min_p``; the token is the first kept one, in
index order, whose running sum of w exceeds u times the kept sum.  A row with
temperature 0 takes the largest logit.  The log probability of the token
among the kept ones comes with it.
"""

import math

import torch

own = False


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one agent decoding: the qkv projection of Qwen2.5-7B, q/k/v adapters of rank 16 stacked
        dict(name="lora_decode_1", op="lora", M=1, K=3584, N=4608, R=48, adapters=4, rows="mixed", bias=True, swiglu=False),
        # a decode batch of 16 agents over 8 roles: the gate/up projection with its SwiGLU
        dict(name="lora_decode_16_swiglu", op="lora", M=16, K=3584, N=37888, R=32, adapters=8, rows="mixed", bias=False, swiglu=True),
        # an odd decode batch, every row one of 32 adapters: the o projection of Qwen3-32B
        dict(name="lora_decode_61", op="lora", M=61, K=8192, N=5120, R=16, adapters=32, rows="mixed", bias=False, swiglu=False),
        # a short prompt on the small test model
        dict(name="lora_prompt_300_small", op="lora", M=300, K=512, N=1024, R=8, adapters=3, rows="runs", bias=True, swiglu=False),
        # the repair rows of a 16K Link: the qkv projection, a few requests in one batch
        dict(name="lora_prompt_5087", op="lora", M=5087, K=3584, N=4608, R=48, adapters=4, rows="runs", bias=True, swiglu=False),
        # a 2048-row prefill batch of several agents: the gate/up projection with its SwiGLU
        dict(name="lora_prompt_2048_swiglu", op="lora", M=2048, K=3584, N=37888, R=128, adapters=6, rows="runs", bias=False, swiglu=True),
        # one agent, the usual chat setting (temperature, top-k 20, top-p 0.8)
        dict(name="sample_1_chat", op="sample", B=1, V=152064, dtype="bf16", mode="chat", pad=0),
        # a decode batch in which every request has settings of its own, greedy ones among them
        dict(name="sample_16_mixed", op="sample", B=16, V=152064, dtype="bf16", mode="mixed", pad=0),
        # 64 requests with top-p alone
        dict(name="sample_64_nucleus", op="sample", B=64, V=151936, dtype="bf16", mode="nucleus", pad=0),
        # many rollouts from the model's own distribution
        dict(name="sample_256_full", op="sample", B=256, V=152064, dtype="bf16", mode="full", pad=0),
        # the small test vocabulary, logits in 32 bits, min-p
        dict(name="sample_7_small_minp", op="sample", B=7, V=2048, dtype="fp32", mode="minp", pad=0),
        # an odd vocabulary in 32 bits (logits that penalties have been added to), rows of a wider buffer
        dict(name="sample_33_odd_mixed", op="sample", B=33, V=50001, dtype="fp32", mode="mixed", pad=7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        M = _log_int(rng, 1, 5000)
        K = 8 * _log_int(rng, 8, 1024)
        swiglu = rng.random() < 0.4
        N = 32 * _log_int(rng, 4, 1024) if swiglu else 8 * _log_int(rng, 16, 4096)
        while M * N * K > 2048 * 37888 * 3584:
            M = (M + 1) // 2
        return dict(op="lora", M=M, K=K, N=N, R=8 * _log_int(rng, 1, 24), adapters=_log_int(rng, 1, 48),
                    rows="mixed" if M <= 128 else "runs", bias=rng.random() < 0.5, swiglu=swiglu)
    V = _log_int(rng, 100, 160000)
    B = _log_int(rng, 1, max(1, min(256, 256 * 152064 // V)))
    return dict(op="sample", B=B, V=V, dtype=rng.choice(["bf16", "fp32"]),
                mode=rng.choice(["chat", "mixed", "nucleus", "full", "minp"]), pad=rng.choice([0, 1, 8]))


# ------------------------------------------------------------------ inputs
def _row_adapters(case, g):
    """Adapter of each row on the host; -1: none."""
    M, n = case["M"], case["adapters"]
    if case["rows"] == "mixed":  # one request a row
        return torch.randint(-1, n, (M,), generator=g) if M > 1 else torch.randint(0, n, (M,), generator=g)
    ids = torch.full((M,), -1, dtype=torch.int64)  # runs of rows, one request each
    at, runs = 0, max(2, min(8, M // 64))
    while at < M:
        length = int(torch.randint(1, 2 * M // runs + 2, (1,), generator=g))
        ids[at:at + length] = int(torch.randint(-1, n, (1,), generator=g))
        at += length
    return ids


def _prepare_lora(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    M, K, N, R, n = (case[k] for k in ("M", "K", "N", "R", "adapters"))

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    rows = _row_adapters(case, h)
    st = {"case": case, "x": normal(M, K), "w": normal(N, K, std=0.02),
          "bias": normal(N, std=0.1) if case["bias"] else None,
          "a": normal(n, R, K, std=K ** -0.5), "b": normal(n, N, R, std=0.05),
          "scale": (0.5 + 2.0 * torch.rand(n, generator=g, device="cuda")), "rows": rows.cuda()}
    if own:
        from sglang_legolink_b200 import ops

        st["lora"] = ops.LoraStack(st["a"], st["b"], st["scale"])
        st["plan"] = ops.lora_plan(rows, "cuda")
    return st


def _settings(case, g):
    """Per-row temperature, top_k, top_p, min_p of a batch's requests."""
    B, mode = case["B"], case["mode"]
    t, k = torch.ones(B), torch.zeros(B, dtype=torch.int32)
    p, m = torch.ones(B), torch.zeros(B)
    if mode == "chat":
        t[:], k[:], p[:] = 0.7, 20, 0.8
    elif mode == "nucleus":
        t[:], p[:] = 0.9, 0.95
    elif mode == "minp":
        m[:] = 0.05
    elif mode == "mixed":
        def pick(values):
            return torch.tensor(values)[torch.randint(0, len(values), (B,), generator=g)]

        t = pick([0.0, 0.6, 0.7, 1.0, 1.3])
        k = pick([0, 0, 1, 20, 50, 1000]).to(torch.int32)
        p = pick([1.0, 0.8, 0.9, 0.95, 0.99])
        m = pick([0.0, 0.0, 0.02, 0.1])
    return t.cuda(), k.cuda(), p.cuda(), m.cuda()


def _prepare_sample(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    B, V = case["B"], case["V"]
    # a heavy upper tail: some rows near-certain, some with thousands of likely tokens
    spread = 0.8 + 1.2 * torch.rand(B, 1, generator=g, device="cuda")
    x = torch.randn(B, V, generator=g, device="cuda") + spread * torch.empty(B, V, device="cuda").exponential_(generator=g)
    wide = torch.zeros(B, V + case["pad"], device="cuda", dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    wide[:, :V] = x
    t, k, p, m = _settings(case, h)
    u = torch.rand(B, generator=h, dtype=torch.float64).cuda()
    return {"case": case, "logits": wide[:, :V], "u": u, "t": t, "k": k, "p": p, "m": m}


def prepare(case, seed):
    return _prepare_lora(case, seed) if case["op"] == "lora" else _prepare_sample(case, seed)


# -------------------------------------------------------------- plain forms
def _plain_lora(st):
    x, a, b = st["x"].float(), st["a"].float(), st["b"].float()
    n, R, K = a.shape
    M, N = x.shape[0], b.shape[1]
    y = x @ st["w"].float().t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    mine = (st["rows"][:, None] == torch.arange(n, device=x.device)).float() * st["scale"]
    s = (x @ a.reshape(n * R, K).t()).view(M, n, R) * mine[:, :, None]
    y = y + s.reshape(M, n * R) @ b.transpose(1, 2).reshape(n * R, N)
    if st["case"]["swiglu"]:
        y = y.view(M, N // 32, 2, 16)
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(M, N // 2)
    return y.to(torch.bfloat16)


def _plain_sample(st):
    # 64 bits: which token a border falls on depends on sums over the whole vocabulary
    x = st["logits"].double()
    B, V = x.shape
    t, p, m = (st[c].double()[:, None] for c in "tpm")
    k = st["k"].long()[:, None]
    top = x.max(dim=1, keepdim=True).values
    greedy = t <= 0
    w = torch.exp((x - top) / torch.where(greedy, torch.ones_like(t), t))
    ws, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = torch.gather(w, 1, order)
    k = torch.where((k <= 0) | (k > V), torch.full_like(k, V), k)
    keep = torch.arange(V, device=x.device)[None, :] < k
    ws = ws * keep
    cum = torch.cumsum(ws, dim=1)
    first = torch.arange(V, device=x.device)[None, :] == 0
    keep &= first | (p >= 1) | (cum - ws < p * cum[:, -1:])
    keep &= ws >= torch.clamp(m, max=1.0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    wk = w * kept
    cum = torch.cumsum(wk, dim=1)
    total = cum[:, -1:]
    ids = (cum > st["u"][:, None] * total).to(torch.uint8).argmax(dim=1, keepdim=True)
    lowest = torch.where(x == top, torch.arange(V, device=x.device)[None, :], V).min(dim=1, keepdim=True).values
    ids = torch.where(greedy, lowest, ids)
    logp = torch.log(torch.gather(w, 1, ids) / total)
    logp = torch.where(greedy, torch.zeros_like(logp), logp)
    return ids[:, 0].to(torch.int32), logp[:, 0].float()


def run(state):
    case = state["case"]
    if own:
        from sglang_legolink_b200 import ops

        if case["op"] == "lora":
            return ops.linear_lora(state["x"], state["w"], state["bias"], state["lora"], state["plan"],
                                   swiglu_epilogue=case["swiglu"])
        return ops.sample(state["logits"], state["u"], state["t"], state["k"], state["p"], state["m"],
                          return_logprobs=True)
    return _plain_lora(state) if case["op"] == "lora" else _plain_sample(state)


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "lora":
        M, K, N, R = (case[k] for k in ("M", "K", "N", "R"))
        used = min(M, case["adapters"])
        out = N // 2 if case["swiglu"] else N
        moved = 2 * (M * K + N * K + M * out + used * R * (K + N) + (N if case["bias"] else 0)) + 4 * (used + M)
        return {"bytes": moved, "flops": 2 * M * (N * K + R * (K + N))}
    size = 2 if case["dtype"] == "bf16" else 4
    B, V = case["B"], case["V"]
    # a subtraction, a product, an exponential and a sum for each logit
    return {"bytes": B * V * size + B * (8 + 16 + 8), "flops": 4 * B * V}


# ------------------------------------------------------------ in 64 bits
def _exact_lora(case, seed):
    st = _prepare_lora(case, seed)
    x = st["x"].to(torch.float64)
    y = torch.matmul(x, st["w"].to(torch.float64).T)
    if st["bias"] is not None:
        y += st["bias"].to(torch.float64)
    for j in range(case["adapters"]):
        rows = torch.nonzero(st["rows"] == j)[:, 0]
        if rows.numel():
            low = torch.matmul(x[rows], st["a"][j].to(torch.float64).T)
            y[rows] += float(st["scale"][j]) * torch.matmul(low, st["b"][j].to(torch.float64).T)
    if not case["swiglu"]:
        return y
    cols = torch.arange(case["N"], device=y.device)
    gate, up = y[:, cols % 32 < 16], y[:, cols % 32 >= 16]
    return gate * torch.sigmoid(gate) * up


def _exact_sample(case, seed):
    st = _prepare_sample(case, seed)
    logp = []
    for b in range(case["B"]):
        x, t = st["logits"][b].to(torch.float64), float(st["t"][b])
        if t <= 0:
            logp.append(0.0)
            continue
        k = int(st["k"][b])
        order = torch.argsort(-x, stable=True)[: k if 0 < k < case["V"] else case["V"]]
        prob = torch.softmax(x[order] / t, dim=0)
        before = torch.cat([prob.new_zeros(1), torch.cumsum(prob, dim=0)[:-1]])
        p = float(st["p"][b])
        count = max(1, int((before < p).sum())) if p < 1 else len(order)
        count = min(count, max(1, int((prob >= min(1.0, float(st["m"][b])) * prob[0]).sum())))
        order, _ = torch.sort(order[:count])  # index order
        prob = torch.softmax(x[order] / t, dim=0)
        at = int(torch.searchsorted(torch.cumsum(prob, dim=0), st["u"][b], right=True))
        logp.append(float(torch.log(prob[min(at, count - 1)])))
    return [None, torch.tensor(logp, dtype=torch.float64)]


def exact(case, seed):
    return _exact_lora(case, seed) if case["op"] == "lora" else _exact_sample(case, seed)
