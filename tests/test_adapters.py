"""Low-rank adapters and the one-launch sampler as the engine runs them:
prefill, Compile, Link and decode of batches that mix adapters, compared with
models whose weights hold the adapter's product."""

import json

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.models.adapters import PROJECTIONS, Adapter
from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import ForwardBatch, QwenModel
from sglang_legolink_b200.ops import reference as ref
from sglang_legolink_b200.runtime.engine import Engine, KernelFault, LinkSourceUnavailable
from sglang_legolink_b200.runtime.sampling import SamplingParams, draw_rows, make_generator, sample_rows
from sglang_legolink_b200.runtime.scheduler import Request, Scheduler

DIMS = {"q_proj": lambda c: (c.hidden_size, c.q_size), "k_proj": lambda c: (c.hidden_size, c.kv_size),
        "v_proj": lambda c: (c.hidden_size, c.kv_size), "o_proj": lambda c: (c.q_size, c.hidden_size),
        "gate_proj": lambda c: (c.hidden_size, c.intermediate_size),
        "up_proj": lambda c: (c.hidden_size, c.intermediate_size),
        "down_proj": lambda c: (c.intermediate_size, c.hidden_size)}


def state_of(cfg, rank, seed, projections=PROJECTIONS, layers=None):
    """PEFT-named random matrices, large enough to change the logits."""
    g = torch.Generator().manual_seed(seed)
    st = {}
    for layer in range(cfg.num_layers) if layers is None else layers:
        for p in projections:
            i, o = DIMS[p](cfg)
            pre = f"base_model.model.model.layers.{layer}.{'mlp' if p in PROJECTIONS[4:] else 'self_attn'}.{p}"
            st[f"{pre}.lora_A.weight"] = (torch.randn(rank, i, generator=g) * i ** -0.5).bfloat16().float()
            st[f"{pre}.lora_B.weight"] = (torch.randn(o, rank, generator=g) * 0.03).bfloat16().float()
    return st


def merged(model, adapter):
    """A CPU fp32 model whose weights hold ``model``'s plus the adapter's."""
    c = model.cfg
    m = QwenModel.random_init(c, seed=0)
    for lw, src in zip(m.layers, model.layers):
        for n in src.__slots__:
            v = getattr(src, n)
            setattr(lw, n, None if v is None else v.float().cpu().clone())
    m.embed, m.final_norm = model.embed.float().cpu(), model.final_norm.float().cpu()
    m.lm_head = m.embed if model.lm_head is model.embed else model.lm_head.float().cpu()
    for i, lw in enumerate(m.layers if adapter is not None else []):
        def delta(p):
            ab = adapter.mats.get((i, p))
            o, k = DIMS[p](c)[1], DIMS[p](c)[0]
            return torch.zeros(o, k) if ab is None else adapter.scale * (ab[1].double() @ ab[0].double()).float()

        lw.qkv_w += torch.cat([delta("q_proj"), delta("k_proj"), delta("v_proj")])
        lw.o_w += delta("o_proj")
        lw.gu_w += ops.interleave_gate_up(delta("gate_proj"), delta("up_proj"))
        lw.down_w += delta("down_proj")
    return m


def adapters_of(cfg):
    return {"one": Adapter.from_state(state_of(cfg, 8, 1), alpha=16, rank=8),
            "two": Adapter.from_state(state_of(cfg, 12, 2, ("q_proj", "v_proj", "up_proj"), range(0, cfg.num_layers, 2)),
                                      alpha=24, rank=12)}


def engine(name="tiny-qwen2", device="cpu", dtype=torch.float32, load=("one", "two"), **kw):
    m = QwenModel.random_init(PRESETS[name], seed=0, device=device, dtype=dtype)
    e = Engine(m, num_pages=1024, page_size=16, max_context=4096, legolink_only=False, **kw)
    ads = adapters_of(m.cfg)
    for n in load:
        e.load_adapter(n, ads[n])
    return e, ads


def toks(n, seed, vocab=1024):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def logits_of(e, prompt, adapter):
    got = {}
    take = e._sample
    e._sample = lambda lo, *a, **k: got.setdefault("l", lo.float().cpu()) is None or take(lo, *a, **k)
    try:
        e.free(e.prefill(prompt, adapter=adapter))
    finally:
        del e._sample
    return got["l"][0]


@pytest.fixture(scope="module")
def world():
    return engine()


@pytest.mark.parametrize("name", ["one", "two"])
def test_prefill_and_decode_equal_the_merged_weights(world, name):
    eng, ads = world
    other = Engine(merged(eng.model, ads[name]), num_pages=512, page_size=16, legolink_only=False)
    p = toks(70, 3)
    a, b, base = logits_of(eng, p, name), logits_of(other, p, None), logits_of(eng, p, None)
    # fp32 on both sides, the products only summed in another order: a few
    # hundred roundings of 2^-24 pass through two layers
    assert (a - b).norm() <= 1e-4 * b.norm()
    assert (a - base).norm() > 100 * 1e-4 * base.norm()  # and the adapter's effect is far above that
    s, f = eng.prefill(p, adapter=name), other.prefill(p)
    eng.decode([s], 10), other.decode([f], 10)
    assert s.output_ids == f.output_ids
    eng.free(s)


def test_a_batch_may_mix_adapters(world):
    eng, _ = world
    names = [None, "one", "two", "one", None]
    alone = []
    for i, n in enumerate(names):
        s = eng.prefill(toks(20 + 7 * i, i), adapter=n)
        eng.decode([s], 6)
        alone.append(list(s.output_ids))
        eng.free(s)
    seqs = [eng.prefill(toks(20 + 7 * i, i), adapter=n) for i, n in enumerate(names)]
    eng.decode(seqs, 6)
    assert [s.output_ids for s in seqs] == alone
    for s in seqs:
        eng.free(s)


def test_compile_and_link_run_with_the_adapter_they_name():
    eng, _ = engine()
    b0, b1, suffix = toks(40, 5), toks(33, 6), toks(9, 7)
    eng.compile(b0, "x", sub_context={"adapter_id": "one"})
    eng.compile_batch([(b1, "y", {"adapter_id": "one"}), (b1, "z")])
    plan = {"cache_keys": ["y", "x"], "recompute_tokens_per_block": [len(b1), len(b0)], "adapter_id": "one"}
    s = eng.link(dict(plan), suffix)
    f = eng.prefill(b1 + b0 + suffix, adapter="one")
    n = eng.prefill(b1 + b0 + suffix)
    eng.decode([s, f, n], 8)
    assert s.output_ids == f.output_ids and n.output_ids != f.output_ids
    # linked rows hold the adapter's K: the first block's equal the prefill's
    lazy = eng.link({**plan, "recompute_tokens_per_block": [0, 0]}, suffix)
    for pos in (0, 17, 32):
        a, b = (eng.kv.k[1][q.pages[pos // 16], :, pos % 16] for q in (lazy, f))
        assert torch.allclose(a, b, atol=1e-4)
    with pytest.raises(LinkSourceUnavailable):  # blocks of one adapter link only under it
        eng.link({"cache_keys": ["y", "x"]}, suffix)
    with pytest.raises(LinkSourceUnavailable):
        eng.link({"cache_keys": ["z"], "adapter_id": "one"}, suffix)


def test_prefix_cache_is_kept_per_adapter(world):
    eng, _ = world
    p = toks(64, 8)
    for n in (None, "one", "two"):
        want = logits_of(eng, p, n)
        for _ in range(2):  # the second finds the first's pages
            s = eng.prefill(p, adapter=n, use_prefix_cache=True, namespace="t")
            assert s.output_ids[0] == int(want.argmax())
            eng.free(s)


def test_a_label_that_names_no_adapter_stays_a_label():
    eng, ads = engine(load=("one",))
    b = toks(32, 9)
    eng.compile(b, "x", sub_context={"adapter_id": "legal"})
    plan = {"cache_keys": ["x"], "recompute_tokens_per_block": [32], "adapter_id": "legal"}
    s, f = eng.link(dict(plan), [1, 2]), eng.prefill(b + [1, 2])
    eng.decode([s, f], 4)
    assert s.output_ids == f.output_ids
    # once an adapter of that name is loaded, its blocks are other blocks
    eng.load_adapter("legal", ads["two"])
    with pytest.raises(LinkSourceUnavailable):
        eng.link(dict(plan), [1, 2])
    eng.compile(b, "y", sub_context={"adapter_id": "legal"})
    s = eng.link({**plan, "cache_keys": ["y"]}, [1, 2])
    f = eng.prefill(b + [1, 2], adapter="legal")
    eng.decode([s, f], 4)
    assert s.output_ids == f.output_ids


def test_the_compatibility_key_names_the_adapters_weights():
    a, _ = engine(load=("one",))
    b, ads = engine(load=())
    plain = b.compat_key("one")
    b.load_adapter("one", ads["two"])
    c, _ = engine(load=("one", "two"))
    assert a.compat_key() == b.compat_key() == c.compat_key() and a.compat_key("x") == b.compat_key("x")
    assert a.compat_key("one") == c.compat_key("one")
    assert len({a.compat_key("one"), b.compat_key("one"), plain}) == 3


def test_requests_reach_their_adapter():
    eng, _ = engine()
    want = eng.prefill(toks(30, 4), adapter="two")
    eng.decode([want], 3)
    sch = Scheduler(eng, legolink_only=False)
    r = sch.submit(Request("plain", "a", toks(30, 4), 4, adapter="two"))
    bad = sch.submit(Request("plain", "b", toks(30, 4), 4, adapter="three"))
    while sch.step():
        pass
    events = [r.events.get_nowait() for _ in range(5)]
    assert [t for kind, t in events if kind == "token"] == want.output_ids and events[4][0] == "done"
    kind, message = bad.events.get_nowait()
    assert kind == "error" and "not loaded" in message


def test_a_checkpoint_directory(tmp_path, world):
    from safetensors.torch import save_file

    eng, ads = world
    st = state_of(eng.cfg, 8, 1)
    save_file(st, str(tmp_path / "adapter_model.safetensors"))
    cfg = {"peft_type": "LORA", "r": 8, "lora_alpha": 16, "bias": "none"}
    (tmp_path / "adapter_config.json").write_text(json.dumps(cfg))
    got = Adapter.from_pretrained(str(tmp_path))
    assert got.scale == ads["one"].scale and got.mats.keys() == ads["one"].mats.keys()
    assert all(torch.equal(got.mats[k][j], ads["one"].mats[k][j]) for k in got.mats for j in (0, 1))
    (tmp_path / "adapter_config.json").write_text(json.dumps({**cfg, "use_rslora": True}))
    assert Adapter.from_pretrained(str(tmp_path)).scale == pytest.approx(16 / 8 ** 0.5)
    for bad in ({"use_dora": True}, {"bias": "all"}, {"rank_pattern": {"q_proj": 4}}, {"peft_type": "IA3"}):
        (tmp_path / "adapter_config.json").write_text(json.dumps({**cfg, **bad}))
        with pytest.raises(ValueError):
            Adapter.from_pretrained(str(tmp_path))


def test_the_service_runs_requests_with_their_adapter(tmp_path):
    from safetensors.torch import save_file

    from sglang_legolink_b200.server.http_server import adapter_arg, build_service

    save_file(state_of(PRESETS["tiny-qwen2"], 8, 1), str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 16}))
    name, path = adapter_arg(f"legal={tmp_path}")
    svc = build_service("tiny-qwen2", max_context=4096, legolink_only=False, sampler="kernel", adapters=[(name, path)])
    try:
        def ask(text, **kw):
            return svc.complete({"messages": [{"role": "user", "content": text}], "max_tokens": 5, "ignore_eos": True,
                                 **kw})["meta_info"]["output_ids"]

        assert ask("a question", adapter_id="legal") != ask("a question")
        sampled = {"temperature": 0.9, "top_p": 0.9, "min_p": 0.02, "seed": 5}
        assert ask("a question", adapter_id="legal", **sampled) == ask("a question", adapter_id="legal", **sampled)
        ask("a block of text " * 8, sub_context={"cache_key": "k", "adapter_id": "legal"})
        linked = ask("and so?", pic_link={"cache_keys": ["k"], "recompute_initial_tokens": 4, "adapter_id": "legal"})
        assert len(linked) == 5
        with pytest.raises(Exception, match="noc_residency_recovery"):
            ask("and so?", pic_link={"cache_keys": ["k"], "recompute_initial_tokens": 4})
        with pytest.raises(Exception, match="not loaded"):
            ask("a question", adapter_id="other")
    finally:
        svc.scheduler.stop()
    for bad in ("legal", "=path", "legal="):
        with pytest.raises(Exception, match="NAME=PATH"):
            adapter_arg(bad)


def test_adapter_refusals(world):
    eng, ads = world
    cfg = eng.cfg
    st = state_of(cfg, 8, 3)
    with pytest.raises(ValueError, match="loaded already"):
        eng.load_adapter("one", ads["two"])
    with pytest.raises(ValueError, match="not a low-rank matrix"):
        Adapter.from_state({"model.embed_tokens.lora_A.weight": torch.zeros(8, 4)}, 8, 8)
    half = dict(st)
    del half[next(k for k in half if "lora_B" in k)]
    with pytest.raises(ValueError, match="do not match"):
        Adapter.from_state(half, 8, 8)
    with pytest.raises(ValueError, match="do not match"):
        Adapter.from_state(st, 8, 16)
    with pytest.raises(ValueError, match="needs a name"):
        eng.load_adapter("", ads["two"])
    with pytest.raises(ValueError, match="exceeds 256"):
        eng.load_adapter("wide", Adapter.from_state(state_of(cfg, 88, 4, ("q_proj", "k_proj", "v_proj")), 8, 88))
    with pytest.raises(ValueError, match="names layers"):
        eng.load_adapter("deep", Adapter.from_state(state_of(cfg, 8, 4, layers=[cfg.num_layers]), 8, 8))
    with pytest.raises(ValueError, match="no matrices"):
        eng.load_adapter("none", Adapter.from_state({}, 8, 8))
    wrong = {k: v[:, :-8] if "lora_A" in k else v for k, v in st.items()}
    with pytest.raises(ValueError, match="do not fit"):
        eng.load_adapter("narrow", Adapter.from_state(wrong, 8, 8))
    nan = {k: torch.full_like(v, float("nan")) for k, v in st.items()}
    with pytest.raises(ValueError, match="finite"):
        eng.load_adapter("nan", Adapter.from_state(nan, 8, 8))
    assert eng.adapters == ["one", "two"]  # a refused adapter leaves nothing behind
    with pytest.raises(ValueError, match="not loaded"):
        eng.prefill([1, 2, 3], adapter="nan")
    shard = QwenModel.random_init(cfg, seed=0, tp_rank=0, tp_size=2)
    with pytest.raises(ValueError, match="tensor parallelism"):
        shard.add_adapter("one", ads["one"])


def test_a_plan_in_use_refuses_an_adapter_behind_its_stack():
    stack = ops.LoraStack(torch.zeros(2, 8, 16), torch.zeros(2, 8, 8), torch.ones(2))
    plan = ops.lora_plan([0, 1, -1], "cpu", max_planes=3)
    ops.linear_lora(torch.zeros(3, 16), torch.zeros(8, 16), None, stack, plan)
    plan.update([1, 1, 0])
    with pytest.raises(ValueError, match="stack of 2"):
        plan.update([0, 2, 1])


# ------------------------------------------------------------------ sampler
def test_min_p_restricts_support():
    logits = torch.tensor([0.5, 0.3, 0.15, 0.05]).log()[None]
    assert SamplingParams.from_request({"temperature": 1, "min_p": 0.4}).min_p == 0.4
    for draw in (sample_rows, draw_rows):
        p = SamplingParams(temperature=1.0, min_p=0.5, seed=0)
        g = [make_generator(p, "cpu")]
        seen = {int(draw(logits, [p], g)[0]) for _ in range(200)}
        assert seen == {0, 1}
        p = SamplingParams(temperature=1.0, min_p=7.0, seed=0)  # beyond 1: the largest
        assert {int(draw(logits, [p], g)[0]) for _ in range(20)} == {0}


def test_drawn_rows_follow_their_own_settings():
    x = torch.randn(4, 500, generator=torch.Generator().manual_seed(1))
    ps = [SamplingParams(), SamplingParams(temperature=0.7, seed=5, top_k=40, top_p=0.9),
          SamplingParams(temperature=1.3, seed=6, min_p=0.02), SamplingParams(temperature=0.7, seed=5, top_k=40, top_p=0.9)]
    ids = draw_rows(x, ps, [make_generator(p, "cpu") for p in ps])
    assert int(ids[0]) == int(x[0].argmax())
    for i in (1, 2, 3):  # alone as in the batch
        assert int(draw_rows(x[i:i + 1], [ps[i]], [make_generator(ps[i], "cpu")])[0]) == int(ids[i])
    u = torch.rand((), dtype=torch.float64, generator=make_generator(ps[1], "cpu"))
    want, _ = ref.sample(x[1:2], u[None], torch.tensor([0.7]), torch.tensor([40], dtype=torch.int32),
                         torch.tensor([0.9]))
    assert int(want[0]) == int(ids[1])


def test_engine_with_the_one_launch_sampler():
    eng, _ = engine(sampler="kernel")
    p = SamplingParams(temperature=1.0, top_p=0.95, min_p=0.01, seed=11)
    t = toks(40, 2)
    runs = []
    for _ in range(2):
        s = eng.prefill(t, sampling=p, adapter="one")
        eng.decode([s], 8)
        runs.append(list(s.output_ids))
        eng.free(s)
    g = eng.prefill(t)
    eng.decode([g], 8)
    a, b = eng.prefill(t), eng.prefill(t, sampling=p, adapter="one")
    eng.decode([a, b], 8)  # a greedy row beside a sampled one
    assert runs[0] == runs[1] == b.output_ids and a.output_ids == g.output_ids
    with pytest.raises(ValueError, match="sampler"):
        Engine(eng.model, num_pages=64, sampler="fast")


def test_a_row_with_nothing_to_draw_is_an_error(monkeypatch):
    eng, _ = engine(sampler="kernel", load=())
    free = eng.alloc.num_free if hasattr(eng.alloc, "num_free") else None
    fwd = eng.model.forward
    monkeypatch.setattr(eng.model, "forward", lambda *a, **k: torch.full_like(fwd(*a, **k), float("nan")))
    with pytest.raises(KernelFault, match="sampling"):
        eng.prefill([1, 2, 3], sampling=SamplingParams(temperature=1.0, seed=1))
    assert free is None or eng.alloc.num_free == free


# ---------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("preset", ["small-qwen2", "small-qwen3"])
def test_gpu_prefill_is_as_near_fp32_as_without_adapters(preset):
    eng, ads = engine(preset, "cuda", torch.bfloat16)
    for n, prompt in (("one", toks(90, 3)), ("two", toks(300, 4)), ("one", toks(1000, 5))):
        err = {}
        for ad in (None, n):
            cpu = Engine(merged(eng.model, ads[ad] if ad else None), num_pages=512, page_size=16, legolink_only=False)
            want = logits_of(cpu, prompt, None)
            err[ad] = float((logits_of(eng, prompt, ad) - want).norm() / want.norm())
        # the same bf16 roundings of activations on both sides, and 16 more
        # bits of the low-rank rows: within twice the plain model's error
        assert err[n] <= 2 * err[None], err


def gpu_seqs(eng, names, sampling=None, n=40):
    return [eng.prefill(toks(n + 9 * i, i), adapter=a, sampling=sampling and sampling[i]) for i, a in enumerate(names)]


def eager_logits(eng, seqs, bucket):
    """The decode forward of ``seqs`` with the graph's row and split counts."""
    ids, pos, slots, pt, kvl = eng._decode_inputs(seqs, bucket, -(-eng.max_context // 16))
    nsplit = ops.decode_splits(bucket, eng.model.hkv, eng.max_context)
    plan = eng._rows_plan([s.adapter for s in seqs] + [-1] * (bucket - len(seqs)), 1)
    fb = ForwardBatch(mode="decode", input_ids=ids.cuda(), positions=pos.cuda(), slots=slots.cuda(),
                      q_indptr=torch.arange(bucket + 1, dtype=torch.int32).cuda(), page_table=pt.cuda(),
                      kv_lens=kvl.cuda(), logit_rows=None, decode_nsplit=nsplit, lora=plan)
    return eng.model.forward(fb, eng.kv)[: len(seqs)].clone()


@pytest.mark.gpu
def test_gpu_graph_replays_with_other_adapters():
    """One captured graph, its plan updated between replays, against an eager
    forward with the same shapes: bit for bit (two sequences with the same
    tokens may still part where two logits tie, if their splits differ)."""
    eng, _ = engine("small-qwen2", "cuda", torch.bfloat16)
    for names in ([None, "one", "two"], ["two", "two", None], ["one", "two", "one", None], [None] * 3, ["two"] * 4):
        seqs = gpu_seqs(eng, names)
        for _ in range(6):
            for s in seqs:
                eng._ensure_capacity(s, s.length + 1)
            want = eager_logits(eng, seqs, 4) if any(names) else None
            out = eng.decode_step(seqs)
            if want is not None:
                assert torch.equal(eng._graphs[("adapters", 4)]["logits"][: len(seqs)], want), names
            for s, t in zip(seqs, out):
                s.output_ids.append(t)
        for s in seqs:
            eng.free(s)
    assert [k for k in eng._graphs if isinstance(k, tuple)] == [("adapters", 4)]


@pytest.mark.gpu
def test_gpu_link_with_an_adapter_equals_its_prefill():
    eng, _ = engine("small-qwen2", "cuda", torch.bfloat16)
    b0, b1, suffix = toks(333, 5), toks(64, 6), toks(21, 7)
    eng.compile(b0, "x", sub_context={"adapter_id": "one"})
    eng.compile(b1, "y", sub_context={"adapter_id": "one"})
    s = eng.link({"cache_keys": ["y", "x"], "recompute_tokens_per_block": [64, 333], "adapter_id": "one"}, suffix)
    f = eng.prefill(b1 + b0 + suffix, adapter="one")
    eng.decode([s], 12), eng.decode([f], 12)
    assert s.output_ids == f.output_ids


@pytest.mark.gpu
def test_gpu_decode_draws_what_the_statement_draws(monkeypatch):
    """Adapters, graph decode and the sampler together: each step's tokens are
    the statement's for that step's logits and the rows' own uniforms."""
    from sglang_legolink_b200.runtime import engine as engine_module

    eng, _ = engine("small-qwen2", "cuda", torch.bfloat16, sampler="kernel")
    ps = [SamplingParams(temperature=0.8, top_p=0.9, seed=1), SamplingParams(), SamplingParams(temperature=1.2, seed=2),
          SamplingParams(temperature=1.0, top_k=20, min_p=0.05, seed=3), SamplingParams(temperature=0.5, top_k=200, seed=4)]
    names = ["one", "two", None, "one", "two"]
    steps = []
    real = draw_rows

    def spy(logits, params, gens, copy):
        state = [None if g is None else g.get_state() for g in gens]
        ids = real(logits, params, gens, copy)
        twins = []
        for st in state:
            t = None
            if st is not None:
                t = torch.Generator()
                t.set_state(st)
            twins.append(t)
        steps.append((ids.cpu(), real(logits.cpu(), params, twins)))
        return ids

    monkeypatch.setattr(engine_module, "draw_rows", spy)
    seqs = gpu_seqs(eng, names, ps)
    eng.decode(seqs, 12)
    assert len(steps) == 4 + 12
    for got, want in steps:
        assert torch.equal(got, want)
    again = gpu_seqs(eng, names, ps)
    eng.decode(again, 12)
    assert [s.output_ids for s in again] == [s.output_ids for s in seqs]
