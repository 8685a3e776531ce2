"""The norm of each head followed by rotary positions in float64, with its gradients from the formulas."""

from __future__ import annotations

import torch

from .rotary import rotary


def qk_norm_rotary(x, weight=None, frequencies=None, eps=1e-6, positions=None, amplitude=1.0, interleaved=False, dy=None):
    """y of x [B, L, H, D], or (y, dx, dweight) for an upstream dy; frequencies: radians per position of each pair, None: no turn."""
    x = x.detach().double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    args = (frequencies, positions, amplitude, interleaved)
    rms = x.square().mean(-1, keepdim=True).add(eps).sqrt()
    h = x / rms
    y = h * w if frequencies is None else rotary(h * w, *args)
    if dy is None:
        return y
    t = dy.detach().double().cpu()
    t = t if frequencies is None else rotary(t, *args, backward=True)
    g = t * w
    return y, (g - h * (g * h).mean(-1, keepdim=True)) / rms, (t * h).sum((0, 1, 2))
