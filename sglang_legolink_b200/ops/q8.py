"""Matrices in 8 bits: e4m3 values with one fp32 scale a row.

``y[m, k]`` stands as ``scale[m] * values[m, k]`` with ``scale[m] = max(amax |y[m]|
/ 448, 2^-126)`` (448 is the largest e4m3 number), so a value is off by half of
an e4m3 step: 2^-4 of itself, or 2^-10 of the scale where it is small.  A row of
a weight ``[N, K]`` is an output feature, a row of an activation a token: both
scales leave the sum over K of a product.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

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
        raise ValueError(f"{name}: values must be [rows, K] with a scale a row, got {tuple(v.shape)}, {tuple(s.shape)}")
    if v.device != s.device:
        raise ValueError(f"{name}: values are on {v.device}, scales on {s.device}")


def check_rows(x, out: Optional[Q8], w, residual, residual_out) -> Q8:
    """Checks of the row operators' arguments; the result to write."""
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, K], got {tuple(x.shape)}")
    K = x.shape[1]
    if K < 16 or K % 16 or K > Q8_MAX_K:
        raise ValueError(f"K must be a multiple of 16, at most {Q8_MAX_K}, got {K}")
    if w is not None and tuple(w.shape) != (K,):
        raise ValueError(f"the norm's weight must be [{K}], got {tuple(w.shape)}")
    for t, name in ((residual, "residual"), (residual_out, "residual_out")):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{name} must be {list(x.shape)}, got {list(t.shape)}")
    if out is None:
        return empty_q8(x.shape[0], K, x.device)
    check_q8(out, "out")
    if out.values.shape != x.shape:
        raise ValueError(f"out must be {list(x.shape)}, got {list(out.values.shape)}")
    return out


def check_product(x: Q8, w: Q8, bias, residual, out, swiglu: bool) -> int:
    """Checks of a product's arguments; the columns of its result."""
    check_q8(x, "x")
    check_q8(w, "w")
    M, K = x.values.shape
    N = w.values.shape[0]
    if w.values.shape[1] != K:
        raise ValueError(f"x has rows of {K} values, w of {w.values.shape[1]}")
    if N < 1 or K < 16 or K % 16 or N % (32 if swiglu else 8):
        raise ValueError(f"K = {K}, N = {N}: K must be a multiple of 16 and N of 8 (of 32: SwiGLU)")
    cols = N // 2 if swiglu else N
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias must be [{N}], got {tuple(bias.shape)}")
    for t, name in ((residual, "residual"), (out, "out")):
        if t is not None and tuple(t.shape) != (M, cols):
            raise ValueError(f"{name} must be [{M}, {cols}], got {tuple(t.shape)}")
    return cols
