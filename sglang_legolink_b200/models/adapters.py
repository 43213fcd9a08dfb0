"""Low-rank adapters (LoRA) for the Qwen projections.

A request names an adapter with ``adapter_id`` (the Compile / Link wire field;
blocks compiled under one adapter link only under the same one).  Adapters are
read from PEFT checkpoints (``adapter_config.json`` +
``adapter_model.safetensors``) and kept stacked per projection
(:class:`~sglang_legolink_b200.ops.LoraStack`), so that a batch may mix them
row by row.  The fused q/k/v and gate/up projections stack their parts' ranks:
an adapter of rank r takes 3r there and 2r here, at most 256.
"""

from __future__ import annotations

import hashlib
import json
import os
import re
from typing import Optional

import torch

from .. import ops

_KEY = re.compile(r"(?:^|\.)layers\.(\d+)\.(?:self_attn|mlp)\.(\w+_proj)\.lora_([AB])(?:\.\w+)?\.weight$")
PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


class Adapter:
    """One adapter: ``mats[(layer, projection)] = (a [r, in], b [out, r])``
    and the factor ``scale`` of their product."""

    def __init__(self, mats: dict, scale: float):
        self.mats, self.scale = mats, float(scale)

    def digest(self) -> str:
        """Names the weights: blocks compiled with an adapter link only where
        the adapter of that name has the same ones."""
        h = hashlib.blake2b(repr(self.scale).encode(), digest_size=8)
        for k in sorted(self.mats):
            for t in self.mats[k]:
                t = t.detach().float().cpu().contiguous()
                h.update(repr((k, tuple(t.shape))).encode())
                h.update(t.numpy().tobytes())
        return h.hexdigest()

    @classmethod
    def from_state(cls, state: dict, alpha: float, rank: int, rslora: bool = False) -> "Adapter":
        """From PEFT tensor names (``...layers.N.self_attn.q_proj.lora_A.weight``)."""
        half: dict = {}
        for name, t in state.items():
            m = _KEY.search(name)
            if m is None or m[2] not in PROJECTIONS:
                raise ValueError(f"adapter tensor '{name}' is not a low-rank matrix of a projection")
            half.setdefault((int(m[1]), m[2]), {})[m[3]] = t
        for k, ab in half.items():
            if set(ab) != {"A", "B"} or any(t.dim() != 2 for t in ab.values()) \
                    or not ab["A"].shape[0] == ab["B"].shape[1] == rank:
                raise ValueError(f"adapter matrices of layer {k[0]} {k[1]} do not match each other and rank {rank}")
        return cls({k: (ab["A"], ab["B"]) for k, ab in half.items()},
                   alpha / (rank ** 0.5 if rslora else rank))

    @classmethod
    def from_pretrained(cls, path: str) -> "Adapter":
        from safetensors.torch import load_file

        with open(os.path.join(path, "adapter_config.json"), encoding="utf-8") as f:
            cfg = json.load(f)
        if cfg.get("peft_type", "LORA") != "LORA" or cfg.get("use_dora") or cfg.get("bias", "none") != "none":
            raise ValueError("only plain LoRA adapters are supported (no DoRA, no biases)")
        if cfg.get("rank_pattern") or cfg.get("alpha_pattern") or cfg.get("modules_to_save"):
            raise ValueError("per-module ranks, per-module alphas and fully trained modules are not supported")
        state = load_file(os.path.join(path, "adapter_model.safetensors"))
        return cls.from_state(state, float(cfg["lora_alpha"]), int(cfg["r"]), bool(cfg.get("use_rslora")))


def _merged(adapters: list, layer: int, parts: list, in_dim: int):
    """The adapters' (a, per-part b) of a fused projection, its parts
    ``(name, rows)`` stacked in the rank; None where no adapter has any."""
    ranks = [sum(ad.mats[(layer, n)][0].shape[0] for n, _ in parts if (layer, n) in ad.mats) for ad in adapters]
    if not any(ranks):
        return None
    rank = -(-max(ranks) // 8) * 8
    if rank > ops.LORA_MAX_RANK:
        raise ValueError(f"layer {layer} {'+'.join(n for n, _ in parts)}: rank {max(ranks)} of the fused projection "
                         f"exceeds {ops.LORA_MAX_RANK}")
    a = torch.zeros(len(adapters), rank, in_dim)
    b = [torch.zeros(len(adapters), rows, rank) for _, rows in parts]
    for i, ad in enumerate(adapters):
        at = 0
        for (name, rows), bp in zip(parts, b):
            if (layer, name) not in ad.mats:
                continue
            ma, mb = ad.mats[(layer, name)]
            r = ma.shape[0]
            if tuple(ma.shape) != (r, in_dim) or tuple(mb.shape) != (rows, r):
                raise ValueError(f"adapter of layer {layer} {name}: a {tuple(ma.shape)}, b {tuple(mb.shape)} do not "
                                 f"fit a projection [{rows}, {in_dim}]")
            a[i, at:at + r] = ma.float()
            bp[i, :, at:at + r] = mb.float()
            at += r
    return a, b


class LayerAdapters:
    """The stacks of one layer's projections (None: no adapter has one)."""

    __slots__ = ("qkv", "o", "gu", "down")

    def __init__(self, cfg, adapters: list, layer: int, device, dtype):
        scale = torch.tensor([ad.scale for ad in adapters])

        def stack(parts, in_dim, join) -> Optional[ops.LoraStack]:
            m = _merged(adapters, layer, parts, in_dim)
            if m is None:
                return None
            a, b = m
            return ops.LoraStack(a.to(device=device, dtype=dtype), join(b).to(device=device, dtype=dtype),
                                 scale.to(device))

        def interleaved(b):
            return torch.stack([ops.interleave_gate_up(g, u) for g, u in zip(b[0], b[1])])

        H, inter = cfg.hidden_size, cfg.intermediate_size
        self.qkv = stack([("q_proj", cfg.q_size), ("k_proj", cfg.kv_size), ("v_proj", cfg.kv_size)], H,
                         lambda b: torch.cat(b, 1))
        self.o = stack([("o_proj", H)], cfg.q_size, lambda b: b[0])
        self.gu = stack([("gate_proj", inter), ("up_proj", inter)], H, interleaved)
        self.down = stack([("down_proj", H)], inter, lambda b: b[0])
