"""Rotary positions in float64 as products of complex numbers."""

from __future__ import annotations

import torch


def rotary(x, frequencies, positions=None, amplitude=1.0, interleaved=False, backward=False):
    """x [B, L, H, D] turned by positions * frequencies (float64 [rot_dim / 2], radians per position)."""
    B, L, H, D = x.shape
    x = x.detach().double().cpu().clone()
    p = torch.arange(L) if positions is None else positions.cpu()
    angle = p.double().expand(B, L)[:, :, None, None] * frequencies.double().cpu()
    z = torch.polar(torch.full_like(angle, amplitude), -angle if backward else angle)
    half = frequencies.numel()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = torch.complex(x[..., a], x[..., b]) * z
    x[..., a], x[..., b] = y.real, y.imag
    return x
