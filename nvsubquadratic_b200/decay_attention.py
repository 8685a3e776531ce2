"""Linear attention with one decay for each head, over whole sequences and for single tokens.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t

A causal sequence mixer of linear cost whose whole past is one ``[Dk, Dv]`` state for each head:
``decay_attention`` runs over prompts and training sequences (forward and backward),
``decay_attention_step`` takes one token of each running request and its state to the next. The
computation runs in ``libhyfft.so`` (``hyfft_decay_forward`` / ``_backward`` / ``_step``), with no
CPU fallback. The reference has no counterpart (its mixers are convolutions, selective scans and
softmax attention).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["decay_attention", "decay_attention_step"]


def _check(q, k, v, log_decay, token: bool):
    rank, form = (3, "[B, heads, D]") if token else (4, "[B, L, heads, D]")
    for name, t in (("q", q), ("k", k), ("v", v)):
        assert t.ndim == rank, f"{name} must be {form}; got {tuple(t.shape)}"
    assert k.shape[:-1] == v.shape[:-1], f"k and v must have the same heads; got {tuple(k.shape)} and {tuple(v.shape)}"
    assert q.shape[:-2] == k.shape[:-2] and q.shape[-1] == k.shape[-1], (
        f"q and k must agree but for their heads; got {tuple(q.shape)} and {tuple(k.shape)}")
    H, Hk = q.shape[-2], k.shape[-2]
    assert H >= 1 and Hk >= 1 and H % Hk == 0, f"key/value heads must divide the query heads; got {Hk} and {H}"
    assert q.shape[-1] >= 1 and v.shape[-1] >= 1, "head sizes must be positive"
    assert tuple(log_decay.shape) == (H,), f"log_decay must be [{H}]; got {tuple(log_decay.shape)}"
    assert log_decay.is_floating_point(), f"log_decay must be a floating type; got {log_decay.dtype}"
    assert q.dtype == k.dtype == v.dtype, f"q, k and v must share a dtype; got {q.dtype}, {k.dtype}, {v.dtype}"
    if q.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"dtype {q.dtype} is not supported (float32, bfloat16, float16)")


def _check_state(name, t, shape):
    assert tuple(t.shape) == shape, f"{name} must be {list(shape)}; got {tuple(t.shape)}"
    assert t.dtype == torch.float32, f"{name} must be float32; got {t.dtype}"


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with its features next to each other (as it is, wherever they already are)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_PLANS: dict = {}


def _plan(q, k, v, scale, dout=None):
    """(descriptor, (forward, saved, backward) workspace bytes) of a call, built once for each set of shapes and strides."""
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), v.shape, v.stride(), scale,
           None if dout is None else dout.stride())
    hit = _PLANS.get(key)
    if hit is None:
        d = _desc(q, k, v, scale, dout)
        hit = (d, _workspaces(d))
        if len(_PLANS) >= 256:
            _PLANS.clear()
        _PLANS[key] = hit
    return hit


def _desc(q, k, v, scale, dout=None) -> _lib.DecayDesc:
    d = _lib.DecayDesc()
    d.batch, d.length = q.shape[0], q.shape[1] if q.ndim == 4 else 1
    d.heads, d.kv_heads, d.dk, d.dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    d.dtype = _lib.DTYPE_CODE[q.dtype]
    d.scale = scale
    for to, t in ((d.q_stride, q), (d.k_stride, k), (d.v_stride, v), (d.o_stride, dout)):
        if t is not None:
            to[0], to[2] = t.stride(0), t.stride(-2)
            to[1] = t.stride(1) if t.ndim == 4 else 0
    return d


def _workspaces(d) -> tuple[int, int, int]:
    f, s, b = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    lib = _lib.load()
    _lib.check(lib.hyfft_decay_workspace_size(ctypes.byref(d), ctypes.byref(f), ctypes.byref(b)), "hyfft_decay_workspace_size")
    _lib.check(lib.hyfft_decay_saved_size(ctypes.byref(d), ctypes.byref(s)), "hyfft_decay_saved_size")
    return f.value, s.value, b.value


def _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state, want_saved):
    """(o, state or None, the tensors as the library read them and what it leaves for the backward)."""
    dev = _lib.require_cuda(q, k, v, log_decay, initial_state, lengths)
    q, k, v = _unit(q), _unit(k), _unit(v)
    g = log_decay.detach().to(torch.float32).contiguous()
    s0 = initial_state.contiguous() if initial_state is not None else None
    B, L, H, Dk = q.shape
    Dv = v.shape[-1]
    o = q.new_empty((B, L, H, Dv))
    state = g.new_empty((B, H, Dk, Dv)) if want_state else None
    saved = None
    if B:
        d, (need, keep, _) = _plan(q, k, v, scale)
        ws = _lib.workspace(need, dev)
        rc = _lib.load().hyfft_decay_forward(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                                             _lib.ptr(lengths), _lib.ptr(s0), o.data_ptr(), _lib.ptr(state),
                                             ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_decay_forward")
        if keep and want_saved:  # without the rest of the workspace, which is as large as the inputs
            saved = ws if keep == need else ws[:keep].clone()
    return o, state, (q, k, v, g, s0, saved)


class _DecayFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, lengths, scale, want_state):
        o, state, read = _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*read, lengths)
        ctx.scale, ctx.decay_dtype = scale, log_decay.dtype
        return o, state

    @staticmethod
    @_lib.no_second_derivative
    def backward(ctx, do, dstate):
        q, k, v, g, s0, saved, lengths = ctx.saved_tensors
        dev = q.device
        want = ctx.needs_input_grad
        B, L, H, Dk = q.shape
        Dv = v.shape[-1]
        none = (None,) * 3
        if do is None and dstate is None:
            return (None,) * 5 + none
        if do is None:
            do = torch.zeros((B, L, H, Dv), dtype=q.dtype, device=dev)
        do = _unit(do.to(q.dtype))
        if dstate is not None:
            dstate = dstate.to(torch.float32).contiguous()
        dq = q.new_empty(q.shape) if want[0] else None
        dk = k.new_empty(k.shape) if want[1] else None
        ds0 = torch.empty_like(s0) if s0 is not None and want[4] else None
        dv = v.new_empty(v.shape) if want[2] or ds0 is not None else None
        dg = torch.empty_like(g) if want[3] else None
        if B == 0:
            return dq, dk, dv, (torch.zeros_like(g).to(ctx.decay_dtype) if want[3] else None), ds0, *none
        d, (_, _, need) = _plan(q, k, v, ctx.scale, do)
        ws = _lib.workspace(need, dev)
        rc = _lib.load().hyfft_decay_backward(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                                              _lib.ptr(lengths), _lib.ptr(s0), _lib.ptr(saved), do.data_ptr(), _lib.ptr(dstate),
                                              _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(dg), _lib.ptr(ds0),
                                              ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_decay_backward")
        return dq, dk, dv if want[2] else None, dg.to(ctx.decay_dtype) if dg is not None else None, ds0, *none


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                    scale: float | None = None, initial_state: torch.Tensor | None = None,
                    lengths: torch.Tensor | None = None, return_state: bool = False):
    """Linear attention over sequences.

    Args:
        q ``[B, L, H, Dk]``, k ``[B, L, Hk, Dk]``, v ``[B, L, Hk, Dv]``: float32, bfloat16 or float16, any
            batch, token and head strides (views into one projection are read in place). Hk divides H:
            query head h reads key/value head ``h // (H // Hk)``. Dk, Dv <= 256.
        log_decay: ``[H]``, the logarithm of each head's decay for one token (0: no decay, ``-inf``: each
            token sees itself alone). It may require a gradient.
        scale: multiplies the outputs; ``Dk ** -0.5`` by default.
        initial_state: float32 ``[B, H, Dk, Dv]``, the state before the first token; zero by default.
        lengths: int32 ``[B]``: tokens from ``lengths[b]`` on are padding. They are neither read nor counted,
            and their outputs and gradients are zero.
        return_state: also return the float32 state after each sequence's last token, from which
            ``decay_attention_step`` or another call goes on.

    Returns ``o [B, L, H, Dv]`` in q's dtype, or ``(o, state)``. Sums and states are float32. An infinity or a NaN
    reaches what the recurrence lets it reach: no earlier token, no other head. First derivatives only.
    """
    _check(q, k, v, log_decay, token=False)
    B, L, H, Dk = q.shape
    if initial_state is not None:
        _check_state("initial_state", initial_state, (B, H, Dk, v.shape[-1]))
    if lengths is not None:
        assert tuple(lengths.shape) == (B,), f"lengths must be [{B}]; got {tuple(lengths.shape)}"
        assert lengths.dtype == torch.int32, f"lengths must be int32; got {lengths.dtype}"
        lengths = lengths.contiguous()
    scale = Dk ** -0.5 if scale is None else float(scale)
    args = (q, k, v, log_decay, initial_state, lengths, scale, bool(return_state))
    if _lib.autograd_sees(*args[:5]):
        o, state = _DecayFunction.apply(*args)
    else:
        o, state, _ = _forward(*args, False)
    return (o, state) if return_state else o


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                         state: torch.Tensor, *, scale: float | None = None, slots: torch.Tensor | None = None,
                         out_state: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each of B running requests; the new states replace the old ones.

    Args:
        q ``[B, H, Dk]``, k ``[B, Hk, Dk]``, v ``[B, Hk, Dv]``, log_decay, scale: as ``decay_attention``.
        state: float32 contiguous ``[N, H, Dk, Dv]``, updated in place.
        slots: int32 ``[B]``, the row of ``state`` that each request owns (no two the same); a slot outside
            ``0 .. N - 1`` marks an idle request, whose output is zero. None: request b owns row b.
        out_state: where the new states go instead, shaped like ``state``; rows that no request owns are
            left as they are.

    Returns ``o [B, H, Dv]``. Inference only: no gradient is recorded.
    """
    _check(q, k, v, log_decay, token=True)
    B, H, Dk = q.shape
    assert state.ndim == 4, f"state must be [N, {H}, {Dk}, {v.shape[-1]}]; got {tuple(state.shape)}"
    N = state.shape[0]
    _check_state("state", state, (N, H, Dk, v.shape[-1]))
    if _lib.autograd_sees(q, k, v, log_decay, state):
        raise NotImplementedError("decay_attention_step records no gradient: call it under torch.no_grad(), "
                                  "or use decay_attention with L = 1")
    out_state = state if out_state is None else out_state
    _check_state("out_state", out_state, tuple(state.shape))
    assert state.is_contiguous() and out_state.is_contiguous(), "the states must be contiguous"
    if slots is not None:
        assert tuple(slots.shape) == (B,), f"slots must be [{B}]; got {tuple(slots.shape)}"
        assert slots.dtype == torch.int32, f"slots must be int32; got {slots.dtype}"
        slots = slots.contiguous()
    else:
        assert N >= B, f"{B} requests need as many states; got {N}"
    dev = _lib.require_cuda(q, k, v, log_decay, state, out_state, slots)
    q, k, v = _unit(q), _unit(k), _unit(v)
    g = log_decay.to(torch.float32).contiguous()
    o = q.new_empty((B, H, v.shape[-1]))
    if B == 0:
        return o
    if N == 0:  # every request is idle
        return o.zero_()
    d, _ = _plan(q, k, v, Dk ** -0.5 if scale is None else float(scale))
    rc = _lib.load().hyfft_decay_step(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                                      _lib.ptr(slots), N, state.data_ptr(), out_state.data_ptr(), o.data_ptr(),
                                      _lib.stream_ptr(dev))
    _lib.check(rc, "hyfft_decay_step")
    return o
