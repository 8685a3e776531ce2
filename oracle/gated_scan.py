"""The gated linear recurrence in float64, token by token, with its gradients from the formulas."""

from __future__ import annotations

import torch


def gated_scan(x, gate, out_gate=None, form="logit", complement=True, initial_state=None, lengths=None, dy=None, dstate=None):
    """(y, state), or (y, state, dx, dgate, dout_gate or None, dinitial_state) for upstream gradients."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, g, o, h0 = f(x), f(gate), f(out_gate), f(initial_state)
    B, L, C = x.shape
    a, u = (torch.sigmoid(g), torch.sigmoid(-g)) if form == "logit" else (torch.exp(g), -torch.expm1(g))
    ends = [L] * B if lengths is None else [min(max(int(n), 0), L) for n in lengths]
    y, state = torch.zeros_like(x), torch.zeros(B, C, dtype=torch.float64)
    seen = torch.zeros(B, L + 1, C, dtype=torch.float64)
    act = torch.ones_like(x) if o is None else o * torch.sigmoid(o)
    for b in range(B):
        h = seen[b, 0] = h0[b] if h0 is not None else torch.zeros(C, dtype=torch.float64)
        for t in range(ends[b]):
            h = a[b, t] * h + (u[b, t] * x[b, t] if complement else x[b, t])
            seen[b, t + 1] = h
            y[b, t] = h * act[b, t]
        state[b] = h
    if dy is None:
        return y, state
    dy = f(dy)
    dx, dg, do, dh0 = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(state)
    for b in range(B):
        c = torch.zeros(C, dtype=torch.float64) if dstate is None else f(dstate)[b]
        for t in range(ends[b] - 1, -1, -1):
            G = dy[b, t] * act[b, t] + c
            c = a[b, t] * G
            dx[b, t] = u[b, t] * G if complement else G
            da = G * (seen[b, t] - x[b, t] if complement else seen[b, t])
            dg[b, t] = da * a[b, t] * (u[b, t] if form == "logit" else 1.0)
            if o is not None:
                s = torch.sigmoid(o[b, t])
                do[b, t] = dy[b, t] * seen[b, t + 1] * s * (1 + o[b, t] * (1 - s))
        dh0[b] = c
    return y, state, dx, dg, do if o is not None else None, dh0
