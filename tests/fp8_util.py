"""Blocks of 8-bit floating point by their definition, in 64 bits and apart from the kernels."""
from __future__ import annotations

import torch


def byte_of(top: torch.Tensor) -> torch.Tensor:
    """The scale's byte of blocks whose largest finite magnitudes are ``top`` (float64): the least e >= -127 with
    top <= 448 * 2^e, as e + 127; 127 for zeros."""
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).clamp_min(-127)
    return (e + 127).to(torch.int64)


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value of finite float64 ``v`` up to 448, ties to even."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def rows(x: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, bytes)`` of ``x [m, k]``: what its blocks stand for (float64; NaN where x is not finite), and the scales'
    bytes ``[ceil(m / block_rows), ceil(k / 128)]``."""
    x = x.double()
    m, k = x.shape
    nb, mb = -(-k // 128), -(-m // block_rows)
    full = torch.zeros((mb * block_rows, nb * 128), dtype=torch.float64, device=x.device)
    full[:m, :k] = x
    fine = torch.where(full.isfinite(), full, 0.0)
    b = byte_of(fine.abs().reshape(mb, block_rows, nb, 128).amax((1, 3)))
    scale = torch.exp2((b - 127).double()).repeat_interleave(block_rows, 0).repeat_interleave(128, 1)
    v = torch.where(full.isfinite(), e4m3(fine / scale) * scale, torch.nan)
    return v[:m, :k], b
