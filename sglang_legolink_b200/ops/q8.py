"""Matrices in 8 bits: e4m3 values with one fp32 scale a row.

``y[m, k]`` stands as ``scale[m] * values[m, k]`` with ``scale[m] = max(amax |y[m]|
/ 448, 2^-126)`` (448 is the largest e4m3 number), so a value is off by half of
an e4m3 step: 2^-4 of itself, or 2^-10 of the scale where it is small.  A row of
a weight ``[N, K]`` is an output feature, a row of an activation a token: both
scales leave the sum over K of a product.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

Q8_MAX_K = 32768  # longest row that is quantised


class Q8(NamedTuple):
    """``values`` [rows, K] (``torch.float8_e4m3fn``) and ``scale`` [rows] (fp32)."""

    values: torch.Tensor
    scale: torch.Tensor

    def float(self) -> torch.Tensor:
        """What it stands for, in fp32."""
        return self.values.float() * self.scale[:, None]


def empty_q8(rows: int, K: int, device) -> Q8:
    return Q8(torch.empty(rows, K, dtype=torch.float8_e4m3fn, device=device),
              torch.empty(rows, dtype=torch.float32, device=device))


def check_q8(t: Q8, name: str) -> None:
    v, s = t
    if v.dtype != torch.float8_e4m3fn or s.dtype != torch.float32:
        raise ValueError(f"{name}: values must be float8_e4m3fn and scales float32, got {v.dtype} and {s.dtype}")
    if v.dim() != 2 or tuple(s.shape) != (v.shape[0],):
        raise ValueError(f"{name}: values must be [rows, K] with a scale a row, got {tuple(v.shape)} and {tuple(s.shape)}")
    if v.device != s.device:
        raise ValueError(f"{name}: values are on {v.device}, scales on {s.device}")


def check_rows(x: torch.Tensor) -> None:
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, K], got {tuple(x.shape)}")
    K = x.shape[1]
    if K < 16 or K % 16 or K > Q8_MAX_K:
        raise ValueError(f"K must be a multiple of 16, at most {Q8_MAX_K}, got {K}")
