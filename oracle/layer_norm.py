"""Layer norm over the last axis in float64, with its gradients from the formulas."""

from __future__ import annotations

import torch


def layer_norm(x, weight=None, bias=None, eps=1e-5, dy=None):
    """y, or (y, dx, dweight, dbias) for an upstream dy."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, w, b = f(x), f(weight), f(bias)
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    h = (x - mean) * rstd
    y = h if w is None else h * w
    y = y if b is None else y + b
    if dy is None:
        return y
    dy = f(dy)
    g = dy if w is None else dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    lead = tuple(range(x.ndim - 1))
    return y, dx, (dy * h).sum(lead), dy.sum(lead)
