"""The one-launch sampler reports a row with nothing to draw (-1) for that row
alone: the sequence of that row fails, its neighbours keep their tokens."""

import pytest
import torch

from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import QwenModel
from sglang_legolink_b200.runtime.engine import Engine, KernelFault
from sglang_legolink_b200.runtime.sampling import SamplingParams
from sglang_legolink_b200.runtime.scheduler import Request, Scheduler

SAMPLED = SamplingParams(temperature=1.0, seed=1)


def engine():
    m = QwenModel.random_init(PRESETS["tiny-qwen2"], seed=0)
    return Engine(m, num_pages=512, page_size=16, max_context=2048, legolink_only=False, sampler="kernel")


def toks(n, seed):
    return torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def spoil(monkeypatch, eng, bad, calls=None):
    """From now on the logits rows that ``bad(batch)`` names are NaN."""
    fwd = eng.model.forward

    def forward(fb, kv, *a, **k):
        out = fwd(fb, kv, *a, **k).clone()
        for r in bad(fb):
            out[r] = float("nan")
        return out

    monkeypatch.setattr(eng.model, "forward", forward)


def test_decode_keeps_the_neighbours(monkeypatch):
    eng = engine()
    alone = []
    for i, sp in enumerate((None, SAMPLED)):
        s = eng.prefill(toks(30, i), sampling=sp)
        eng.decode([s], 6)
        alone.append(list(s.output_ids))
        eng.free(s)
    free = eng.alloc.num_free
    a, bad, b = eng.prefill(toks(30, 0)), eng.prefill(toks(20, 9), sampling=SAMPLED), eng.prefill(toks(30, 1), sampling=SAMPLED)
    spoil(monkeypatch, eng, lambda fb: [i for i, n in enumerate(fb.kv_lens.tolist()) if n < 27])
    out = eng.decode_step([a, bad, b])
    assert out[1] == -1 and isinstance(bad.error, KernelFault) and bad.finished
    assert a.error is None and b.error is None and out[0] == alone[0][1] and out[2] == alone[1][1]
    for s, t in ((a, out[0]), (b, out[2])):
        s.output_ids.append(t)
    with pytest.raises(KernelFault):  # it stays failed, and is refused before anything runs
        eng.decode_step([a, bad])
    assert a.length == 31
    eng.decode([a, bad, b], 5)  # the others go on
    assert a.output_ids == alone[0] and b.output_ids == alone[1] and -1 not in bad.output_ids
    for s in (a, bad, b):
        eng.free(s)
    assert eng.alloc.num_free == free


def test_engine_decode_reports_the_row_after_the_others_are_done(monkeypatch):
    eng = engine()
    want = eng.prefill(toks(30, 0))
    eng.decode([want], 6)
    a, bad = eng.prefill(toks(30, 0)), eng.prefill(toks(20, 9), sampling=SAMPLED)
    spoil(monkeypatch, eng, lambda fb: [i for i, n in enumerate(fb.kv_lens.tolist()) if n < 24])
    with pytest.raises(KernelFault, match="sampling"):
        eng.decode([a, bad], 6)
    assert a.output_ids == want.output_ids and bad.error is not None and -1 not in bad.output_ids


def test_an_extend_step_fails_the_one_link(monkeypatch):
    eng = engine()
    eng.compile(toks(32, 5), "x")
    plan = {"cache_keys": ["x"], "recompute_tokens_per_block": [4]}
    want = eng.link(dict(plan), [1, 2], sampling=SAMPLED)
    first = list(want.output_ids)
    eng.free(want)
    free = eng.alloc.num_free
    spoil(monkeypatch, eng, lambda fb: [1])
    c, links = eng.extend_step(compiles=[(toks(40, 6), "y")], links=[(dict(plan), [1, 2], None, SAMPLED),
                                                                     (dict(plan), [1, 2], None, SAMPLED)])
    assert c[0]["cache_key"] == "y"
    assert isinstance(links[0], KernelFault) and "sampling" in str(links[0])
    assert links[1].output_ids == first
    eng.free(links[1])
    assert free - eng.alloc.num_free == 3  # the compiled block's own pages


def test_the_scheduler_fails_one_request(monkeypatch):
    eng = engine()
    sch = Scheduler(eng, legolink_only=False)
    good = sch.submit(Request("plain", "a", toks(30, 0), 6))
    bad = sch.submit(Request("plain", "b", toks(20, 9), 6, sampling=SAMPLED))
    free = eng.alloc.num_free
    spoil(monkeypatch, eng, lambda fb: [i for i, n in enumerate(fb.kv_lens.tolist()) if n == 22])
    while sch.step():
        pass
    got = [good.events.get_nowait() for _ in range(7)]
    assert [k for k, _ in got] == ["token"] * 6 + ["done"]
    events = []
    while not bad.events.empty():
        events.append(bad.events.get_nowait())
    assert [k for k, _ in events] == ["token", "token", "error"] and "sampling" in events[2][1]
    assert all(t >= 0 for k, t in events if k == "token")
    assert eng.alloc.num_free == free and not sch.running


def test_what_the_two_samplers_keep_where_logits_tie_at_the_border_of_top_k():
    from sglang_legolink_b200.runtime.sampling import draw_rows, make_generator, sample_rows

    x = torch.tensor([[3.0, 1.0, 2.0, 1.0, 1.0, 0.0]])
    p = SamplingParams(temperature=1.0, top_k=3, seed=2)
    for draw, kept in ((sample_rows, {0, 1, 2, 3, 4}), (draw_rows, {0, 1, 2})):
        g = [make_generator(p, "cpu")]
        assert {int(draw(x, [p], g)[0]) for _ in range(600)} == kept
