"""Adding an adapter touches that adapter alone: what is loaded already is not
merged again, no more than one projection's stack exists twice, and an adapter
that cannot be added leaves the others as they were."""

import weakref

import pytest
import torch

from sglang_legolink_b200 import ops
from sglang_legolink_b200.models.adapters import PROJECTIONS, Adapter
from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import QwenModel

CFG = PRESETS["tiny-qwen2"]
H, INTER, Q, KV = CFG.hidden_size, CFG.intermediate_size, CFG.q_size, CFG.kv_size
DIMS = dict(zip(PROJECTIONS, ((H, Q), (H, KV), (H, KV), (Q, H), (H, INTER), (H, INTER), (INTER, H))))
PARTS = {"qkv": ("q_proj", "k_proj", "v_proj"), "o": ("o_proj",), "gu": ("gate_proj", "up_proj"), "down": ("down_proj",)}


def adapter(seed, rank, projections=PROJECTIONS, layers=range(CFG.num_layers)):
    g = torch.Generator().manual_seed(seed)
    return Adapter({(i, p): (torch.randn(rank, DIMS[p][0], generator=g), torch.randn(DIMS[p][1], rank, generator=g))
                    for i in layers for p in projections}, 0.25 + seed)


def model(dtype=torch.float32):
    return QwenModel.random_init(CFG, seed=0, dtype=dtype)


def products(m, layer, name):
    """What the stack of a projection computes for each adapter: scale b a, part by part."""
    st = getattr(m._layer_adapters[layer], name)
    if st is None:
        return None
    out = st.scale[:, None, None].double() * (st.b.double() @ st.a.double())
    if name == "gu":
        n = out.shape[0]
        v = out.view(n, -1, 2, 16, H)
        out = torch.cat([v[:, :, 0].reshape(n, INTER, H), v[:, :, 1].reshape(n, INTER, H)], 1)
    return out


def wanted(adapters, layer, name):
    if not any((layer, p) in ad.mats for ad in adapters for p in PARTS[name]):
        return None
    return torch.stack([torch.cat([ad.scale * (ad.mats[(layer, p)][1].double() @ ad.mats[(layer, p)][0].double())
                                   if (layer, p) in ad.mats else torch.zeros(DIMS[p][1], DIMS[p][0]).double()
                                   for p in PARTS[name]]) for ad in adapters])


def check(m, adapters):
    for layer in range(CFG.num_layers):
        for name in PARTS:
            got, want = products(m, layer, name), wanted(adapters, layer, name)
            assert (got is None) == (want is None), (layer, name)
            # fp32 matrices on both sides: the same values, multiplied in 64 bits; the scale is held in fp32
            assert want is None or torch.allclose(got, want, rtol=1e-6, atol=1e-6), (layer, name)


def several():
    return [adapter(1, 8, ("q_proj", "v_proj")), adapter(2, 12), adapter(3, 4, ("up_proj", "o_proj"), [1]),
            adapter(4, 20, ("down_proj", "k_proj"), [0])]


def test_adapters_of_different_ranks_and_projections_added_one_by_one():
    m, ads = model(), several()
    for i, ad in enumerate(ads):
        assert m.add_adapter(f"a{i}", ad) == i
        check(m, ads[: i + 1])


def test_what_is_loaded_is_not_merged_again():
    m, ads = model(), several()
    kept = several()
    for i, ad in enumerate(ads):
        m.add_adapter(f"a{i}", ad)
        ad.mats.clear()  # nothing needs its matrices any more
    check(m, kept)


def test_one_projection_at_most_exists_twice(monkeypatch):
    live, peak = weakref.WeakSet(), 0
    size = lambda s: s.a.numel() + s.b.numel()  # noqa: E731
    init = ops.LoraStack.__init__

    def counted(self, *a, **k):
        nonlocal peak
        init(self, *a, **k)
        live.add(self)
        peak = max(peak, sum(map(size, live)))

    monkeypatch.setattr(ops.LoraStack, "__init__", counted)
    m = model()
    for i in range(4):
        m.add_adapter(f"a{i}", adapter(i, 8))
        peak = 0
    m.add_adapter("last", adapter(9, 8))
    total, largest = sum(map(size, live)), max(map(size, live))
    assert peak <= total + largest


def test_an_adapter_that_cannot_be_added_leaves_the_others(monkeypatch):
    m, ads = model(), several()
    m.add_adapter("a0", ads[0])
    for bad in (adapter(5, 96), Adapter({**ads[1].mats, (1, "o_proj"): (torch.zeros(12, Q - 1), torch.zeros(H, 12))}, 1.0),
                Adapter({**ads[1].mats, (1, "down_proj"): (torch.full((12, INTER), float("inf")), torch.zeros(H, 12))}, 1.0),
                Adapter(ads[1].mats, float("nan"))):
        with pytest.raises(ValueError):
            m.add_adapter("bad", bad)
        assert m.adapter_names == ["a0"]
        check(m, ads[:1])
    # it runs out of memory in the middle: those that ran before still run, and a second try is a whole one
    join, calls = ops.LoraStack.joined, []

    def fails(self, *a):
        calls.append(1)
        if len(calls) > 3:
            raise torch.OutOfMemoryError("no memory")
        return join(self, *a)

    generation = m.buf_generation
    monkeypatch.setattr(ops.LoraStack, "joined", fails)
    m.add_adapter("a1", adapter(7, 8, ("q_proj",), [0]))  # one call
    with pytest.raises(torch.OutOfMemoryError):
        m.add_adapter("a2", ads[1])
    monkeypatch.setattr(ops.LoraStack, "joined", join)
    assert m.adapter_names == ["a0", "a1"] and m.buf_generation > generation + 1  # captured graphs point at stacks that are gone
    m.add_adapter("a2", ads[1])
    check(m, [ads[0], adapter(7, 8, ("q_proj",), [0]), ads[1]])


def test_a_matrix_that_overflows_the_projections_type_is_refused():
    m = QwenModel.random_init(CFG, seed=0, dtype=torch.bfloat16)
    ad = adapter(1, 8, ("o_proj",), [0])
    ad.mats[(0, "o_proj")][0][0, 0] = 3.4e38  # finite in fp32, infinite in bf16
    with pytest.raises(ValueError, match="finite"):
        m.add_adapter("a", ad)
    assert m.adapter_names == []
