"""Plain forms of the 8-bit operators, on the CPU: quantisation in float32 (every step is one correctly rounded operation, so the
kernels have to give the same bits) and everything else in float64."""

from __future__ import annotations

import torch

FP8 = torch.float8_e4m3fn
EPS32 = 2.0 ** -24            # the largest error of one rounding to float32, relative


def groups(n: int) -> int:
    return (n + 127) // 128


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    s = amax / 448.0
    return torch.where(s < 2.0 ** -126, torch.full_like(s, 2.0 ** -126), s)        # (NaN stays NaN)


def spread(s: torch.Tensor, rows: int, columns: int, block_rows: int) -> torch.Tensor:
    return s[torch.arange(rows) // block_rows][:, torch.arange(columns) // 128]


def quantize(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(values e4m3, scales) of a float32 matrix."""
    R, C = x.shape
    down = R if block_rows == 1 else groups(R)
    s = torch.empty((down, groups(C)))
    for i in range(down):
        for j in range(groups(C)):
            s[i, j] = x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128].abs().max()
    s = scale_of(s)
    v = x * spread(1.0 / s, R, C, block_rows)
    return v.clamp(-448.0, 448.0).to(FP8), s


def values(q: torch.Tensor, s: torch.Tensor, block_rows: int) -> torch.Tensor:
    """What a quantised matrix stands for, in float64."""
    return q.cpu().float().double() * spread(s.cpu().double(), *q.shape, block_rows)


def product(x, xs, w, ws) -> tuple[torch.Tensor, torch.Tensor]:
    """(x @ w^T, bound of a float evaluation's error) in float64.  A term is exact in float (two four-bit significands); it meets at most
    127 others of its group, then the groups' sums meet, each time rounded or cut to a float (a whole unit, 2 EPS32), and three
    roundings more bring the scales in."""
    X, W = values(x, xs, 1), values(w, ws, 128)
    y = X @ W.t()
    steps = 128 + groups(x.shape[1]) + 3
    return y, steps * 2 * EPS32 * (X.abs() @ W.abs().t())


def half_step(v: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The largest error of rounding v to dtype."""
    return v.abs() * (torch.finfo(dtype).eps / 2)


def quantized_error(v: torch.Tensor, s: torch.Tensor, error: torch.Tensor) -> torch.Tensor:
    """The largest distance between v and value * scale of a matrix quantised from v + error (s: its scales): the value is off by
    half a step of e4m3 (2^-4 of it, 2^-10 under the smallest normal), multiplications by s and 1 / s add a few roundings."""
    S = spread(s.cpu().double(), *v.shape, 1)
    return error + ((v.abs() + error) * 2.0 ** -4 + S * 2.0 ** -10) * (1 + 8 * EPS32) + v.abs() * 8 * EPS32
