"""Low-rank adapters of many requests beside one shared projection: the
weights of a projection's adapters and the plan of a batch's rows.

A batch is cut into tiles of rows (one tile for up to 128 rows, 256-row tiles
beyond); each tile has one *plane* per adapter that its rows use.  The kernels
write a plane of low-rank rows per adapter, zero in the rows of other
adapters, and multiply each plane with its adapter's B.
"""

from __future__ import annotations

from typing import Callable, Optional, Sequence, Union

import numpy as np
import torch

LORA_MAX_RANK = 256


class LoraStack:
    """The adapters of one projection ``[N, K]``: ``a`` [n, R, K] and ``b``
    [n, N, R] in the projection's dtype, ``scale`` [n] (alpha / rank).

    R is a multiple of 8, at most 256; a smaller adapter fills its remaining
    rows of ``a`` and columns of ``b`` with zeros (:meth:`stack` does that).
    Where ``w`` is a fused product (q/k/v, interleaved gate/up) the adapters
    of its parts are stacked in R, with ``b`` block-diagonal over the parts.
    The weights must be finite: rows of other adapters in the same tile
    multiply ``b`` with zeros, which would turn an infinity into NaN."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, _checked: int = 0):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"adapter shapes: a {tuple(a.shape)}, b {tuple(b.shape)}")
        n, rank, _ = a.shape
        if n < 1 or rank < 8 or rank % 8 or rank > LORA_MAX_RANK:
            raise ValueError(f"{n} adapters of rank {rank}: the rank must be a multiple of 8, at most {LORA_MAX_RANK}")
        if tuple(scale.shape) != (n,):
            raise ValueError(f"scale must be [{n}], got {tuple(scale.shape)}")
        if a.dtype != b.dtype or a.device != b.device or scale.device != a.device:
            raise ValueError("a, b and scale must share a device, a and b a dtype")
        self.a, self.b = a.contiguous(), b.contiguous()
        self.scale = scale.float().contiguous()
        self.count, self.rank = n, rank
        if not bool(torch.stack([torch.isfinite(t[_checked:]).all() for t in (self.a, self.b, self.scale)]).all()):
            raise ValueError("adapter weights must be finite")

    @classmethod
    def stack(cls, pairs: Sequence[tuple[torch.Tensor, torch.Tensor]], scales: Sequence[float]) -> "LoraStack":
        """Adapters ``(a [r, K], b [N, r])`` of different ranks."""
        rank = -(-max(p[0].shape[0] for p in pairs) // 8) * 8
        a = torch.stack([torch.nn.functional.pad(p[0], (0, 0, 0, rank - p[0].shape[0])) for p in pairs])
        b = torch.stack([torch.nn.functional.pad(p[1], (0, rank - p[1].shape[1])) for p in pairs])
        return cls(a, b, torch.tensor(list(scales), dtype=torch.float32, device=a.device))

    def joined(self, a: torch.Tensor, b: torch.Tensor, scale: float, keep: Optional[int] = None) -> "LoraStack":
        """A stack of this one's adapters (its first ``keep``) and one more,
        ``a`` [r, K] and ``b`` [N, r], as the last; r = 0 for one that leaves
        the projection as it is."""
        n = self.count if keep is None else keep
        r = a.shape[0]
        rank = max(self.rank, -(-r // 8) * 8)
        if a.shape[1:] != self.a.shape[2:] or tuple(b.shape) != (self.b.shape[1], r):
            raise ValueError(f"adapter shapes: a {tuple(a.shape)}, b {tuple(b.shape)}")
        na = self.a.new_zeros(n + 1, rank, self.a.shape[2])
        nb = self.b.new_zeros(n + 1, self.b.shape[1], rank)
        na[:n, : self.rank], nb[:n, :, : self.rank] = self.a[:n], self.b[:n]
        na[n, :r], nb[n, :, :r] = a.to(na), b.to(nb)
        return LoraStack(na, nb, torch.cat([self.scale[:n], self.scale.new_full((1,), scale)]), n)


class LoraPlan:
    """Which adapter each row of a batch uses (:func:`lora_plan`).  One plan
    serves every projection of a forward, on any stream."""

    def __init__(self, row_adapters, device, max_planes: Optional[int] = None,
                 copy: Optional[Callable[[np.ndarray], torch.Tensor]] = None):
        ids = _host_ids(row_adapters)
        self.rows = len(ids)
        self.tile_rows = 128 if self.rows <= 128 else 256
        self.tiles = -(-self.rows // self.tile_rows)
        self.device = torch.device(device)
        self.limit = 1 << 31  # the smallest stack that the plan has been used with
        host, planes = self._build(ids)
        self.max_planes = max(1, planes if max_planes is None else int(max_planes))
        if planes > self.max_planes:
            raise ValueError(f"the rows need {planes} planes, max_planes is {self.max_planes}")
        self._copy = copy
        self.buf: Optional[torch.Tensor] = None
        self._store(ids, host)

    def _build(self, ids: np.ndarray):
        """(row slots, tile offsets, plane keys) and the plane count."""
        tile = np.arange(self.rows, dtype=np.int64) // self.tile_rows
        live = ids >= 0
        # one key per (tile, adapter): planes in tile order, adapters ascending
        keys, inverse = np.unique((tile[live] << 32) | ids[live], return_inverse=True)
        ptr = np.searchsorted(keys, np.arange(self.tiles + 1, dtype=np.int64) << 32)
        slot = np.full(self.rows, -1, dtype=np.int64)
        slot[live] = inverse.reshape(-1) - ptr[tile[live]]
        return (slot, ptr, keys), len(keys)

    def _store(self, ids: np.ndarray, host) -> None:
        slot, ptr, keys = host
        flat = np.zeros(self.rows + self.tiles + 1 + 2 * self.max_planes, dtype=np.int32)
        flat[: self.rows] = slot
        flat[self.rows : self.rows + self.tiles + 1] = ptr
        planes = flat[self.rows + self.tiles + 1 :].reshape(2, self.max_planes)
        planes[0, : len(keys)] = keys & 0xFFFFFFFF
        planes[1, : len(keys)] = keys >> 32
        if self.buf is None:
            self.buf = self._copy(flat) if self._copy else torch.from_numpy(flat).to(self.device)
        else:
            self.buf.copy_(self._copy(flat) if self._copy else torch.from_numpy(flat))
        self.top_adapter = int(ids.max()) if self.rows else -1
        self.row_adapters = torch.from_numpy(ids)

    def update(self, row_adapters) -> "LoraPlan":
        """Gives the same rows other adapters, in the same device buffer: a
        CUDA graph captured with this plan replays with the new ones.  The
        copy is made on the current stream: the one the plan is used on.  Build
        the plan with ``max_planes`` = the most adapters it may ever hold
        (times the row tiles); more than that is refused."""
        ids = _host_ids(row_adapters)
        if len(ids) != self.rows:
            raise ValueError(f"the plan is for {self.rows} rows, got {len(ids)}")
        host, planes = self._build(ids)
        if planes > self.max_planes:
            raise ValueError(f"the rows need {planes} planes, the plan holds {self.max_planes}")
        if ids.size and ids.max() >= self.limit:  # a captured call would read behind its stack
            raise ValueError(f"adapter {int(ids.max())}: the plan was used with a stack of {self.limit}")
        self._store(ids, host)
        return self


def _host_ids(row_adapters) -> np.ndarray:
    if isinstance(row_adapters, torch.Tensor):
        row_adapters = row_adapters.detach().cpu().numpy()
    raw = np.asarray(row_adapters)
    ids = raw.astype(np.int64).reshape(-1)
    if raw.ndim != 1 or (raw.size and not np.array_equal(ids, raw)):
        raise ValueError("row_adapters must be one whole number a row")
    if ids.size and (ids.min() < -1 or ids.max() >= 1 << 31):
        raise ValueError("adapter numbers start at 0; -1: no adapter")
    return ids


def lora_plan(row_adapters: Union[Sequence[int], np.ndarray, torch.Tensor], device,
              max_planes: Optional[int] = None,
              copy: Optional[Callable[[np.ndarray], torch.Tensor]] = None) -> LoraPlan:
    """Plan of a batch whose row m uses adapter ``row_adapters[m]`` (-1: none),
    in any order; host values (a CUDA tensor is read back).  ``copy``: host
    array -> new tensor on ``device``, in place of a copy that the host waits
    for; the plan is then ready on the stream that ``copy`` used."""
    return LoraPlan(row_adapters, device, max_planes, copy)
