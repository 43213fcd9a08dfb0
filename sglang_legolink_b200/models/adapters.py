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


# the projections of a layer's stacks: of each part its name and (in, out) sizes
def _stacks(cfg) -> dict:
    H, inter = cfg.hidden_size, cfg.intermediate_size
    return {"qkv": (("q_proj", H, cfg.q_size), ("k_proj", H, cfg.kv_size), ("v_proj", H, cfg.kv_size)),
            "o": (("o_proj", cfg.q_size, H),),
            "gu": (("gate_proj", H, inter), ("up_proj", H, inter)),
            "down": (("down_proj", inter, H),)}


def check_adapter(cfg, adapter: Adapter, dtype) -> None:
    """Raises ValueError where the adapter does not fit the model, before
    anything of it is on the device."""
    if not torch.isfinite(torch.tensor(adapter.scale, dtype=torch.float32)):
        raise ValueError("adapter weights must be finite")
    for parts in _stacks(cfg).values():
        for layer in range(cfg.num_layers):
            rank = 0
            for name, in_dim, rows in parts:
                if (layer, name) not in adapter.mats:
                    continue
                ma, mb = adapter.mats[(layer, name)]
                r = ma.shape[0]
                if tuple(ma.shape) != (r, in_dim) or tuple(mb.shape) != (rows, r):
                    raise ValueError(f"adapter of layer {layer} {name}: a {tuple(ma.shape)}, b {tuple(mb.shape)} do not "
                                     f"fit a projection [{rows}, {in_dim}]")
                if not (torch.isfinite(ma.to(dtype)).all() and torch.isfinite(mb.to(dtype)).all()):
                    raise ValueError("adapter weights must be finite")
                rank += r
            if rank > ops.LORA_MAX_RANK:
                raise ValueError(f"layer {layer} {'+'.join(n for n, *_ in parts)}: rank {rank} of the fused projection "
                                 f"exceeds {ops.LORA_MAX_RANK}")


def _merged(adapter: Adapter, layer: int, parts):
    """The adapter's (a, per-part b) of a fused projection, its parts stacked
    in the rank."""
    mats = [adapter.mats.get((layer, name)) for name, *_ in parts]
    rank = sum(m[0].shape[0] for m in mats if m is not None)
    a = torch.zeros(rank, parts[0][1])
    b = [torch.zeros(rows, rank) for _, _, rows in parts]
    at = 0
    for m, bp in zip(mats, b):
        if m is not None:
            r = m[0].shape[0]
            a[at:at + r], bp[:, at:at + r] = m[0].float(), m[1].float()
            at += r
    return a, b


class LayerAdapters:
    """The stacks of one layer's projections (None: no adapter has one)."""

    __slots__ = ("qkv", "o", "gu", "down")

    def __init__(self):
        self.qkv: Optional[ops.LoraStack] = None
        self.o: Optional[ops.LoraStack] = None
        self.gu: Optional[ops.LoraStack] = None
        self.down: Optional[ops.LoraStack] = None

    def add(self, cfg, adapter: Adapter, layer: int, keep: int, device, dtype) -> None:
        """Puts an adapter behind the first ``keep``, one projection after the
        other, so that one at most exists twice."""
        for slot, parts in _stacks(cfg).items():
            old = getattr(self, slot)
            a, b = _merged(adapter, layer, parts)
            rank = a.shape[0]
            if old is None and not rank:
                continue
            b = ops.interleave_gate_up(*b) if slot == "gu" and rank else torch.cat(b)
            if old is None:  # the adapters before have none
                padded = -(-rank // 8) * 8
                na = torch.zeros(keep + 1, padded, a.shape[1], device=device, dtype=dtype)
                nb = torch.zeros(keep + 1, b.shape[0], padded, device=device, dtype=dtype)
                na[keep, :rank], nb[keep, :, :rank] = a.to(na), b.to(nb)
                scale = torch.zeros(keep + 1, device=device)
                scale[keep] = adapter.scale
                new = ops.LoraStack(na, nb, scale)
            else:
                new = old.joined(a, b, adapter.scale, keep)
            setattr(self, slot, new)
