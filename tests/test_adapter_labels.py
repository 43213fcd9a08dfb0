"""Adapter ids that name no loaded adapter are free-form labels: none of them
may give the compatibility key of an adapter, or of other request fields."""

import pytest
import torch

from sglang_legolink_b200.models.adapters import PROJECTIONS, Adapter
from sglang_legolink_b200.models.config import PRESETS
from sglang_legolink_b200.models.qwen import QwenModel
from sglang_legolink_b200.runtime.engine import Engine, LinkSourceUnavailable


def engine():
    m = QwenModel.random_init(PRESETS["tiny-qwen2"], seed=0)
    e = Engine(m, num_pages=256, page_size=16, max_context=1024, legolink_only=False)
    c = m.cfg
    g = torch.Generator().manual_seed(1)
    mats = {(0, PROJECTIONS[0]): (torch.randn(8, c.hidden_size, generator=g), torch.randn(c.q_size, 8, generator=g))}
    e.load_adapter("one", Adapter(mats, 1.0))
    return e


def test_no_label_has_the_key_of_a_loaded_adapter():
    e = engine()
    digest = e.model.adapter_digests[0]
    key = e.compat_key("one")
    assert digest in key
    field = key[key.index("adapter_id=") + len("adapter_id="):].split("|")[0]
    for label in (field, f"one#{digest}", f"one%23{digest}", "one%", "one%25"):
        assert e._adapter(label) < 0 and e.compat_key(label) != key
    labels = ["a", "a#b", "a%23b", "a%2523b", "a|b", "a%7Cb", "a%", "a%25", "one", "none#", ""]
    assert len({e.compat_key(x) for x in labels}) == len(labels)


def test_a_field_cannot_run_into_the_next_one():
    e = engine()
    a = e.compat_key("x|attention_backend_fingerprint=y", None, None)
    assert a.count("|") == e.compat_key("x").count("|")
    assert e.compat_key("x", "p|q", "r") != e.compat_key("x", "p", "q|r")
    # ordinary ids stay as they are
    assert "adapter_id=legal-v1|" in e.compat_key("legal-v1")


def test_a_block_compiled_under_a_look_alike_label_does_not_link_as_the_adapters():
    e = engine()
    block = list(range(20, 52))
    label = "one#" + e.model.adapter_digests[0]
    e.compile(block, "x", sub_context={"adapter_id": label})  # the base model's K and V
    with pytest.raises(LinkSourceUnavailable):
        e.link({"cache_keys": ["x"], "recompute_tokens_per_block": [4], "adapter_id": "one"}, [1, 2])
    e.free(e.link({"cache_keys": ["x"], "recompute_tokens_per_block": [4], "adapter_id": label}, [1, 2]))


@pytest.mark.parametrize("none", ["", None])
def test_an_empty_adapter_id_names_no_adapter_in_any_request(none, tmp_path):
    """As in Compile and Link requests, whose key for it is that of no adapter."""
    import json

    from safetensors.torch import save_file

    from sglang_legolink_b200.server.http_server import build_service

    c = PRESETS["tiny-qwen2"]
    pre = "base_model.model.model.layers.0.self_attn.q_proj"
    save_file({f"{pre}.lora_A.weight": torch.randn(8, c.hidden_size), f"{pre}.lora_B.weight": torch.randn(c.q_size, 8)},
              str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 16}))
    svc = build_service("tiny-qwen2", max_context=1024, legolink_only=False, adapters=[("legal", str(tmp_path))])
    try:
        ask = {"messages": [{"role": "user", "content": "a question"}], "max_tokens": 4, "ignore_eos": True}
        want = svc.complete(ask)["meta_info"]["output_ids"]
        assert svc.complete({**ask, "adapter_id": none})["meta_info"]["output_ids"] == want
        eng = svc.scheduler.engine
        assert eng.compat_key(none) == eng.compat_key()
    finally:
        svc.scheduler.stop()
