"""Models whose projections are in 8 bits, in the engine and the service.

Tolerance of the logits against the model's own plain statement: both take the
same roundings, but a sum that differs in its last bits may round to the next
e4m3 value, 2^-3 of one of a row's K >= 256 values; a product then moves by about
2^-3 / sqrt(256) of one typical term, its row by less than 1 % of its norm.
"""

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import ForwardBatch, QwenModel
from sglang_legolink_b200.ops import Q8
from sglang_legolink_b200.ops import reference as ref
from sglang_legolink_b200.runtime.engine import Engine, LinkSourceUnavailable

gpu = pytest.mark.gpu


def tokens(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def statement(m, toks, ranks=()):
    """Logits of the last token: every product on quantised rows, in 64 bits.
    ``ranks``: the shards of a tensor-parallel model (``m`` is its first),
    whose row-parallel products are sums of the ranks' own."""
    c, D = m.cfg, m.cfg.head_dim
    dbl = lambda t: t.detach().cpu().double()  # noqa: E731

    def product(x, w, bias=None):
        q, s = ref.quantize_q8(x.float())
        y = (q.double() * s.double()[:, None]) @ (dbl(w.values.float()) * dbl(w.scale)[:, None]).t()
        return y if bias is None else y + dbl(bias)

    def norm(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + c.rms_norm_eps) * dbl(w)

    ranks = ranks or (m,)
    n = len(toks)
    r = dbl(m.embed)[torch.tensor(toks)]
    cos, sin = dbl(m.cos_sin)[:n].chunk(2, -1)
    mask = torch.full((n, n), float("-inf"), dtype=torch.float64).triu(1)
    def attention(m, lw, h):
        qkv = product(h, lw.qkv_w, lw.qkv_b).view(n, -1, D)
        q, k, v = qkv[:, : m.hq], qkv[:, m.hq : m.hq + m.hkv], qkv[:, m.hq + m.hkv :]
        if lw.q_norm is not None:
            q, k = norm(q, lw.q_norm), norm(k, lw.k_norm)

        def rope(t):
            a, b = t.chunk(2, -1)
            return torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], -1)

        q, k = rope(q), rope(k).repeat_interleave(m.hq // m.hkv, 1)
        v = v.repeat_interleave(m.hq // m.hkv, 1)
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) * m.scale + mask, -1)
        return product(torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1), lw.o_w)

    def mlp(lw, h):
        gu = product(h, lw.gu_w).view(n, -1, 2, 16)
        g, u = gu[:, :, 0], gu[:, :, 1]
        return product((g * torch.sigmoid(g) * u).reshape(n, -1), lw.down_w)

    for i, lw in enumerate(m.layers):
        h = norm(r, lw.in_norm)
        r = r + sum(attention(s, s.layers[i], h) for s in ranks)
        h = norm(r, lw.post_norm)
        r = r + sum(mlp(s.layers[i], h) for s in ranks)
    return norm(r, m.final_norm)[-1] @ torch.cat([dbl(s.lm_head) for s in ranks])[: c.vocab_size].t()


def logits_of(eng, toks):
    pages = eng.alloc.alloc((len(toks) + eng.page_size - 1) // eng.page_size)
    fb = eng._extend_batch([(toks, list(range(len(toks))), pages, len(toks))])
    return eng.model.forward(fb, eng.kv)[-1].float().cpu()


def close(a, b, tol):
    return float((a.double() - b.double()).norm() / b.double().norm()) <= tol


def test_the_forward_follows_its_statement():
    cfg = PRESETS["tiny-qwen2"]
    m = QwenModel.random_init(cfg, seed=3)
    m.quantize_weights()
    assert all(isinstance(getattr(lw, n), Q8) for lw in m.layers for n in ("qkv_w", "o_w", "gu_w", "down_w"))
    toks = tokens(40, cfg.vocab_size, 1)
    assert close(logits_of(Engine(m, num_pages=64, max_context=256), toks), statement(m, toks), 0.02)


def _rank(rank, port, q):
    import os

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    import torch.distributed as dist

    from sglang_legolink_b200.parallel.tp import NcclTPComm

    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        cfg = PRESETS["tiny-qwen2"]
        m = QwenModel.random_init(cfg, seed=3, tp_rank=rank, tp_size=2, comm=NcclTPComm())
        m.quantize_weights()
        eng = Engine(m, num_pages=64, max_context=256)
        toks = tokens(40, cfg.vocab_size, 1)
        pages = eng.alloc.alloc(3)
        fb = eng._extend_batch([(toks, list(range(40)), pages, 40)])
        logits = m.full_logits(m.forward(fb, eng.kv))[-1]
        seq = eng.prefill(toks)
        eng.decode([seq], 4)
        q.put((rank, logits.tolist(), seq.output_ids))
    finally:
        dist.destroy_process_group()


def test_two_tensor_parallel_ranks_follow_their_statement():
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    [p.start() for p in procs]
    got = {r: (logits, ids) for r, logits, ids in (q.get(timeout=300) for _ in procs)}
    [p.join(timeout=60) for p in procs]
    assert all(p.exitcode == 0 for p in procs) and got[0][1] == got[1][1]
    cfg = PRESETS["tiny-qwen2"]
    shards = [QwenModel.random_init(cfg, seed=3, tp_rank=r, tp_size=2) for r in range(2)]
    [m.quantize_weights() for m in shards]
    assert close(torch.tensor(got[0][0]), statement(shards[0], tokens(40, cfg.vocab_size, 1), shards), 0.02)


def test_a_capture_sees_the_parts_and_changes_little(tmp_path):
    from sglang_legolink_b200.runtime.repair_diagnostics import COMPONENTS, RepairStateCapture

    cfg = PRESETS["tiny-qwen2"]
    m = QwenModel.random_init(cfg, seed=3)
    m.quantize_weights()
    eng = Engine(m, num_pages=64, max_context=256)
    toks = tokens(24, cfg.vocab_size, 2)
    plain = logits_of(eng, toks)
    m.capture = RepairStateCapture(tmp_path / "s.pt", range(cfg.num_layers))
    seen = logits_of(eng, toks)
    assert close(seen, plain, 0.02)
    assert all(set(m.capture.component_outputs[i]) == set(COMPONENTS) and i in m.capture.layer_outputs
               for i in range(cfg.num_layers))


def test_refusals(tmp_path):
    cfg = PRESETS["tiny-qwen2"]
    m = QwenModel.random_init(cfg)
    m.layers[1].o_w[3, 4] = float("nan")
    with pytest.raises(ValueError, match="layer 1"):
        m.quantize_weights()
    assert not m.quantized and isinstance(m.layers[0].qkv_w, torch.Tensor)
    m = QwenModel.random_init(cfg.with_(hidden_size=264, num_heads=4, head_dim=66))
    with pytest.raises(ValueError, match="8 bits"):
        m.quantize_weights()
    m = QwenModel.random_init(cfg)
    Engine(m, num_pages=64, max_context=256)
    with pytest.raises(ValueError, match="engine"):
        m.quantize_weights()
    m = QwenModel.random_init(cfg)
    m.quantize_weights()
    m.quantize_weights()  # it is already
    with pytest.raises(ValueError, match="adapters"):
        m.add_adapter("a", None)


def test_blocks_of_other_weights_do_not_link():
    cfg = PRESETS["tiny-qwen2"]
    engines = []
    for q in (False, True):
        m = QwenModel.random_init(cfg)
        if q:
            m.quantize_weights()
        engines.append(Engine(m, num_pages=64, max_context=256))
    assert engines[0].compat_key() != engines[1].compat_key()
    b = engines[1]
    b.compile(tokens(32, cfg.vocab_size, 1), "k")
    seq = b.link({"cache_keys": ["k"], "recompute_initial_tokens": 4}, [1, 2, 3])
    b.decode([seq], 4)
    assert len(seq.output_ids) == 5
    b.compat["model_fingerprint"] = engines[0].compat["model_fingerprint"]  # as an engine of the other weights asks
    with pytest.raises(LinkSourceUnavailable):
        b.link({"cache_keys": ["k"], "recompute_initial_tokens": 4}, [1, 2, 3])


def test_the_service_with_weights_in_8_bits():
    from sglang_legolink_b200.server.http_server import build_service

    svc = build_service("tiny-qwen2", max_context=1024, legolink_only=False, weights="q8")
    try:
        assert svc.scheduler.engine.model.quantized
        ask = {"messages": [{"role": "user", "content": "a question"}], "max_tokens": 5, "ignore_eos": True}
        assert len(svc.complete(dict(ask))["meta_info"]["output_ids"]) == 5
    finally:
        svc.scheduler.stop()


def test_the_command_line_refuses_what_does_not_go_together(capsys):
    from sglang_legolink_b200.server.http_server import main

    for more in (["--adapter", "a=b"], ["--weights", "q4"]):
        with pytest.raises(SystemExit):
            main(["--weights", "q8", *more])
        assert "--weights" in capsys.readouterr().err


# ----------------------------------------------------------------- on the GPU
def small(name="small-qwen2", seed=0, **kw):
    m = QwenModel.random_init(PRESETS[name], seed=seed, device="cuda", dtype=torch.bfloat16)
    m.quantize_weights()
    return Engine(m, num_pages=2048, page_size=16, max_context=8192, **kw)


@gpu
@pytest.mark.parametrize("name", ["small-qwen2", "small-qwen3"])
@pytest.mark.parametrize("n", [1, 17, 90, 300])
def test_the_forward_follows_its_statement_on_the_gpu(name, n):
    """bf16 between the products: 2^-8 of the residual, rotated rows, the attention's and the gated rows."""
    eng = small(name)
    toks = tokens(n, eng.cfg.vocab_size, n)
    assert close(logits_of(eng, toks), statement(eng.model, toks), 0.05)
    assert ops.check_errors("cuda") == 0


@gpu
@pytest.mark.parametrize("name", ["small-qwen2", "small-qwen3"])
def test_a_link_with_every_row_repaired_equals_a_prefill(name):
    eng = small(name)
    subs = [tokens(n, eng.cfg.vocab_size, n) for n in (128, 333, 64, 700)]
    suffix = tokens(21, eng.cfg.vocab_size, 9)
    for i, s in enumerate(subs):
        eng.compile(s, f"k{i}")
    order = [2, 0, 3, 1]
    seq = eng.link({"cache_keys": [f"k{i}" for i in order], "recompute_tokens_per_block": [len(subs[i]) for i in order]},
                   suffix)
    eng.decode([seq], 16)
    full = eng.prefill(sum((subs[i] for i in order), []) + suffix)
    eng.decode([full], 16)
    assert seq.output_ids == full.output_ids


@gpu
def test_decode_in_a_graph_equals_eager_steps():
    eng = small(seed=1)
    prompts = [tokens(n, eng.cfg.vocab_size, n) for n in (5, 40, 130)]
    graph = [eng.prefill(p) for p in prompts]
    eng.decode(graph, 12)
    eng.use_cuda_graphs = False
    eager = [eng.prefill(p) for p in prompts]
    eng.decode(eager, 12)
    assert [s.output_ids for s in graph] == [s.output_ids for s in eager]


@gpu
def test_decode_step_equals_the_prefill_of_the_same_tokens():
    """The last row of a prefill and a decode step take other kernels and splits: close, not the same bits."""
    eng = small(seed=2)
    toks = tokens(50, eng.cfg.vocab_size, 4)
    want = logits_of(eng, toks)
    pages = eng.alloc.alloc(4)
    fb = eng._extend_batch([(toks[:-1], list(range(49)), pages, 49)])
    eng.model.forward(fb, eng.kv)
    dev = eng.device
    fb = ForwardBatch(mode="decode", input_ids=torch.tensor(toks[-1:], dtype=torch.int32, device=dev),
                      positions=torch.tensor([49], dtype=torch.int32, device=dev),
                      slots=torch.tensor([pages[3] * 16 + 1], dtype=torch.int64, device=dev),
                      q_indptr=torch.tensor([0, 1], dtype=torch.int32, device=dev),
                      page_table=torch.tensor([pages], dtype=torch.int32, device=dev),
                      kv_lens=torch.tensor([50], dtype=torch.int32, device=dev))
    got = eng.model.forward(fb, eng.kv)[0].float().cpu()
    assert close(got, want, 0.05)


@pytest.mark.parametrize("which", ["FFN", "OUTPUT_PROJECTION"])
def test_a_setting_of_row_wise_repair_is_refused_ahead_of_the_first_request(monkeypatch, capsys, which):
    """It acts on grouped Compiles alone: a server that starts with it would fail under load."""
    from sglang_legolink_b200.server.http_server import build_service, main

    name = "SGLANG_PIC_SPARSE_REPAIR_ROWWISE_" + which
    ready = QwenModel.random_init(PRESETS["tiny-qwen2"])
    ready.quantize_weights()
    monkeypatch.setenv(name, "1")
    m = QwenModel.random_init(PRESETS["tiny-qwen2"])
    with pytest.raises(ValueError, match=name):
        m.quantize_weights()
    assert not m.quantized and isinstance(m.layers[0].qkv_w, torch.Tensor)
    with pytest.raises(ValueError, match=name):
        Engine(ready, num_pages=64, max_context=256)
    with pytest.raises(ValueError, match=name):
        build_service("tiny-qwen2", max_context=1024, legolink_only=False, weights="q8")
    with pytest.raises(SystemExit):
        main(["--weights", "q8"])
    assert name in capsys.readouterr().err
    Engine(m, num_pages=64, max_context=256)  # as before for the other weights
    monkeypatch.setenv(name, "0")
    Engine(ready, num_pages=64, max_context=256)


def test_an_engine_that_was_not_made_holds_nothing():
    """An engine whose arguments do not fit leaves the model as it was."""
    m = QwenModel.random_init(PRESETS["tiny-qwen2"])
    for bad in (dict(page_size="16"), dict(max_blocks="many"), dict(num_pages="64")):
        with pytest.raises((TypeError, ValueError)):
            Engine(m, **{"num_pages": 64, "max_context": 256, **bad})
    m.quantize_weights()
    assert m.quantized


def test_the_service_refuses_weights_that_it_does_not_know():
    from sglang_legolink_b200.server.http_server import build_service

    with pytest.raises(ValueError, match="weights"):
        build_service("tiny-qwen2", max_context=1024, legolink_only=False, weights="fp8")
