"""Linear attention with one decay for each head, token by token in float64, with its gradients from the
formulas (nothing here is differentiated automatically).

    S_t = a S_{t-1} + k_t v_t^T,  o_t = scale * S_t^T q_t,  a = exp(log_decay[h])
    G_t = dL/dS_t = a G_{t+1} + scale * q_t do_t^T  (dL/dS_L added at a sequence's last token)
    dq_t = scale * S_t do_t,  dk_t = G_t v_t,  dv_t = G_t^T k_t,  dS_0 = a G_1
    T_t = dS_t / dlog_decay = a (T_{t-1} + S_{t-1}),  dlog_decay = sum_t scale * q_t^T T_t do_t + <dS_L, T_L>
"""

from __future__ import annotations

import torch


def _prep(q, k, v, log_decay, lengths, initial_state):
    B, L, H, Dk = q.shape
    r = H // k.shape[2]
    f = lambda t: t.detach().double().cpu()  # noqa: E731
    q, k, v = f(q), f(k).repeat_interleave(r, 2), f(v).repeat_interleave(r, 2)
    n = lengths.cpu().long().clamp(0, L) if lengths is not None else torch.full((B,), L)
    a = torch.exp(f(log_decay))[None, :, None, None].expand(B, H, 1, 1)
    S = f(initial_state).clone() if initial_state is not None else torch.zeros(B, H, Dk, v.shape[-1], dtype=torch.float64)
    return q, k, v, n, a, S


def decay_attention(q, k, v, log_decay, scale=None, initial_state=None, lengths=None):
    """(o, state) in float64."""
    B, L, H, Dk = q.shape
    scale = Dk ** -0.5 if scale is None else scale
    q, k, v, n, a, S = _prep(q, k, v, log_decay, lengths, initial_state)
    o = torch.zeros(B, L, H, v.shape[-1], dtype=torch.float64)
    for t in range(L):
        on = n > t
        S[on] = a[on] * S[on] + torch.einsum("bhk,bhv->bhkv", k[on, t], v[on, t])
        o[on, t] = scale * torch.einsum("bhk,bhkv->bhv", q[on, t], S[on])
    return o, S


def decay_attention_grads(q, k, v, log_decay, do, dstate=None, scale=None, initial_state=None, lengths=None):
    """(dq, dk, dv, dlog_decay, dinitial_state) in float64."""
    B, L, H, Dk = q.shape
    Hk = k.shape[2]
    scale = Dk ** -0.5 if scale is None else scale
    q, k, v, n, a, S = _prep(q, k, v, log_decay, lengths, initial_state)
    do = do.detach().double().cpu()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    T = torch.zeros_like(S)
    dg = torch.zeros(H, dtype=torch.float64)
    for t in range(L):
        on = n > t
        T[on] = a[on] * (T[on] + S[on])
        S[on] = a[on] * S[on] + torch.einsum("bhk,bhv->bhkv", k[on, t], v[on, t])
        dq[on, t] = scale * torch.einsum("bhkv,bhv->bhk", S[on], do[on, t])
        dg += scale * torch.einsum("bhk,bhkv,bhv->h", q[on, t], T[on], do[on, t])
    U = torch.zeros_like(S)  # what reaches a state from behind
    if dstate is not None:
        U = dstate.detach().double().cpu().clone()
        dg += torch.einsum("bhkv,bhkv->h", U, T)
    for t in reversed(range(L)):
        on = n > t
        G = U[on] + scale * torch.einsum("bhk,bhv->bhkv", q[on, t], do[on, t])
        dk[on, t] = torch.einsum("bhkv,bhv->bhk", G, v[on, t])
        dv[on, t] = torch.einsum("bhkv,bhk->bhv", G, k[on, t])
        U[on] = a[on] * G
    shared = lambda x: x.view(B, L, Hk, H // Hk, x.shape[-1]).sum(3)  # noqa: E731
    return dq, shared(dk), shared(dv), dg, U
