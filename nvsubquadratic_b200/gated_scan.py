"""Gated linear recurrence: every channel keeps a running mean (or sum) whose memory each token sets for itself.

    a_t = sigmoid(gate_t)  or  exp(gate_t)
    h_t = a_t h_{t-1} + (1 - a_t) x_t  or  a_t h_{t-1} + x_t,    y_t = h_t  or  h_t * silu(out_gate_t)

``gated_scan`` runs over prompts and training sequences (forward and backward) in one pass over the data,
``gated_scan_step`` takes one token of each running request and its state to the next. Where ``decay_attention`` keeps
a matrix for each head under one constant decay, this keeps one number for each channel under decays that the
tokens choose. The computation runs in ``libhyfft.so`` (``hyfft_gated_forward`` / ``_backward`` / ``_step``), with no
CPU fallback. The reference's recurrent mixer (``nvsubquadratic/modules/mamba_nd.py``) calls an external selective scan.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["gated_scan", "gated_scan_step"]

_FORM_CODE = {"logit": 0, "log": 1}


def _check(x, gate, out_gate, form, token: bool):
    rank, shape = (2, "[B, C]") if token else (3, "[B, L, C]")
    assert x.ndim == rank and x.shape[-1] >= 1, f"x must be {shape}; got {tuple(x.shape)}"
    for name, t in (("gate", gate), ("out_gate", out_gate)):
        if t is not None:
            assert t.shape == x.shape, f"{name} must be {list(x.shape)} as x; got {tuple(t.shape)}"
            assert t.dtype == x.dtype, f"x and {name} must share a dtype; got {x.dtype} and {t.dtype}"
    if form not in _FORM_CODE:
        raise ValueError(f"unknown form {form!r}: use 'logit' or 'log'")
    if x.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"dtype {x.dtype} is not supported (float32, bfloat16, float16)")


def _check_state(name, t, shape):
    assert tuple(t.shape) == shape, f"{name} must be {list(shape)}; got {tuple(t.shape)}"
    assert t.dtype == torch.float32, f"{name} must be float32; got {t.dtype}"


def _unit(t: torch.Tensor | None) -> torch.Tensor | None:
    """t with its channels next to each other (as it is, wherever they already are)."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_PLANS: dict = {}


def _plan(x, gate, out_gate, form, complement, dy=None):
    """(descriptor, bytes kept for the backward) of a call, built once for each set of shapes and strides."""
    key = (x.shape, x.stride(), x.dtype, gate.stride(), None if out_gate is None else out_gate.stride(), form, complement,
           None if dy is None else dy.stride())
    hit = _PLANS.get(key)
    if hit is None:
        d = _lib.GatedDesc()
        d.batch, d.channels, d.length = x.shape[0], x.shape[-1], x.shape[1] if x.ndim == 3 else 1
        d.dtype, d.form, d.complement = _lib.DTYPE_CODE[x.dtype], _FORM_CODE[form], int(complement)
        for to, t in ((d.x_stride, x), (d.gate_stride, gate), (d.out_gate_stride, out_gate), (d.dy_stride, dy)):
            if t is not None:  # the stride of an axis of one entry is not used, and may be anything
                to[0] = t.stride(0) if t.shape[0] > 1 else 0
                to[1] = t.stride(1) if t.ndim == 3 and t.shape[1] > 1 else 0
        size = ctypes.c_size_t()
        _lib.check(_lib.load().hyfft_gated_saved_size(ctypes.byref(d), ctypes.byref(size)), "hyfft_gated_saved_size")
        hit = (d, size.value)
        if len(_PLANS) >= 256:
            _PLANS.clear()
        _PLANS[key] = hit
    return hit


def _forward(x, gate, out_gate, initial_state, lengths, form, complement, want_state, keep):
    """(y, state or None, the tensors as the library read them and what it keeps for the backward)."""
    dev = _lib.require_cuda(x, gate, out_gate, initial_state, lengths)
    x, gate, out_gate = _unit(x), _unit(gate), _unit(out_gate)
    h0 = initial_state.contiguous() if initial_state is not None else None
    B, L, C = x.shape
    y = x.new_empty(x.shape)
    state = x.new_empty((B, C), dtype=torch.float32) if want_state else None
    saved = None
    if B and L:
        d, size = _plan(x, gate, out_gate, form, complement)
        if keep:
            saved = _lib.workspace(size, dev)
        rc = _lib.load().hyfft_gated_forward(ctypes.byref(d), x.data_ptr(), gate.data_ptr(), _lib.ptr(out_gate),
                                             _lib.ptr(lengths), _lib.ptr(h0), y.data_ptr(), _lib.ptr(state), _lib.ptr(saved),
                                             size if keep else 0, _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_gated_forward")
    elif want_state:  # no tokens
        state.copy_(h0) if h0 is not None else state.zero_()
    return y, state, (x, gate, out_gate, saved)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, out_gate, initial_state, lengths, form, complement, want_state):
        y, state, read = _forward(x, gate, out_gate, initial_state, lengths, form, complement, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*read, lengths)
        ctx.args = (form, complement)
        return y, state

    @staticmethod
    @_lib.no_second_derivative
    def backward(ctx, dy, dstate):
        x, gate, out_gate, saved, lengths = ctx.saved_tensors
        none = (None,) * 4
        if dy is None and dstate is None:
            return (None,) * 4 + none
        want = ctx.needs_input_grad
        B, L, C = x.shape
        dstate = dstate.to(torch.float32).contiguous() if dstate is not None else None
        dh0 = x.new_empty((B, C), dtype=torch.float32) if want[3] else None
        dx, dg = x.new_empty(x.shape), x.new_empty(x.shape)
        do = x.new_empty(x.shape) if out_gate is not None else None
        if B == 0 or L == 0:
            if dh0 is not None:
                dh0.copy_(dstate) if dstate is not None else dh0.zero_()
        else:
            dy = x.new_zeros(x.shape) if dy is None else _unit(dy.to(x.dtype))
            d, size = _plan(x, gate, out_gate, *ctx.args, dy)
            rc = _lib.load().hyfft_gated_backward(ctypes.byref(d), x.data_ptr(), gate.data_ptr(), _lib.ptr(out_gate),
                                                  _lib.ptr(lengths), saved.data_ptr(), size, dy.data_ptr(),
                                                  _lib.ptr(dstate), dx.data_ptr(), dg.data_ptr(), _lib.ptr(do),
                                                  _lib.ptr(dh0), _lib.stream_ptr(x.device))
            _lib.check(rc, "hyfft_gated_backward")
        return dx if want[0] else None, dg if want[1] else None, do if want[2] else None, dh0, *none


def gated_scan(x: torch.Tensor, gate: torch.Tensor, *, out_gate: torch.Tensor | None = None, form: str = "logit",
               complement: bool = True, initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
               return_state: bool = False):
    """The recurrence over sequences.

    Args:
        x, gate, out_gate ``[B, L, C]``: float32, bfloat16 or float16, any batch and token strides (views into one
            projection, and expanded batches, are read in place).
        form: what ``gate`` holds. ``"logit"``: the decay is its sigmoid; ``"log"``: its exponential (0 and below for
            a recurrence that forgets, ``-inf``: each token sees itself alone).
        complement: weigh each token by ``1 - a_t`` (the state stays within the range of the inputs) or by 1.
        out_gate: multiplies the outputs by ``silu(out_gate)``.
        initial_state: float32 ``[B, C]``, the state before the first token; zero by default.
        lengths: int32 ``[B]``: tokens from ``lengths[b]`` on are padding. They are neither read nor counted,
            and their outputs and gradients are zero.
        return_state: also return the float32 state after each sequence's last token, from which
            ``gated_scan_step`` or another call goes on.

    Returns ``y [B, L, C]`` in x's dtype, or ``(y, state)``. Sums and states are float32, ``1 - a`` is computed without
    cancellation. Decays above 1 are taken as they are: what float32 holds of a growing state comes out; decays below 2^-126 are
    0. An infinity or a NaN reaches what the recurrence lets it reach: no earlier token, no other channel. First
    derivatives only.
    """
    _check(x, gate, out_gate, form, token=False)
    B, L, C = x.shape
    if initial_state is not None:
        _check_state("initial_state", initial_state, (B, C))
    if lengths is not None:
        assert tuple(lengths.shape) == (B,), f"lengths must be [{B}]; got {tuple(lengths.shape)}"
        assert lengths.dtype == torch.int32, f"lengths must be int32; got {lengths.dtype}"
        lengths = lengths.contiguous()
    args = (x, gate, out_gate, initial_state, lengths, form, bool(complement), bool(return_state))
    if _lib.autograd_sees(x, gate, out_gate, initial_state):
        y, state = _GatedScan.apply(*args)
    else:
        y, state, _ = _forward(*args, False)
    return (y, state) if return_state else y


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, out_gate: torch.Tensor | None = None,
                    form: str = "logit", complement: bool = True, slots: torch.Tensor | None = None,
                    out_state: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each of B running requests; the new states replace the old ones.

    Args:
        x, gate, out_gate ``[B, C]``, form, complement: as ``gated_scan``.
        state: float32 contiguous ``[N, C]``, updated in place.
        slots: int32 ``[B]``, the row of ``state`` that each request owns (no two the same); a slot outside
            ``0 .. N - 1`` marks an idle request, whose output is zero and whose input is not read. None: request b owns row b.
        out_state: where the new states go instead, shaped like ``state``; rows that no request owns are
            left as they are.

    Returns ``y [B, C]``. Inference only: no gradient is recorded.
    """
    _check(x, gate, out_gate, form, token=True)
    B, C = x.shape
    assert state.ndim == 2, f"state must be [N, {C}]; got {tuple(state.shape)}"
    N = state.shape[0]
    _check_state("state", state, (N, C))
    if _lib.autograd_sees(x, gate, out_gate, state):
        raise NotImplementedError("gated_scan_step records no gradient: call it under torch.no_grad(), "
                                  "or use gated_scan with L = 1")
    out_state = state if out_state is None else out_state
    _check_state("out_state", out_state, (N, C))
    assert state.is_contiguous() and out_state.is_contiguous(), "the states must be contiguous"
    if slots is not None:
        assert tuple(slots.shape) == (B,), f"slots must be [{B}]; got {tuple(slots.shape)}"
        assert slots.dtype == torch.int32, f"slots must be int32; got {slots.dtype}"
        slots = slots.contiguous()
    else:
        assert N >= B, f"{B} requests need as many states; got {N}"
    dev = _lib.require_cuda(x, gate, out_gate, state, out_state, slots)
    x, gate, out_gate = _unit(x), _unit(gate), _unit(out_gate)
    y = x.new_empty((B, C))
    if B == 0:
        return y
    if N == 0:  # every request is idle
        return y.zero_()
    d, _ = _plan(x, gate, out_gate, form, bool(complement))
    rc = _lib.load().hyfft_gated_step(ctypes.byref(d), x.data_ptr(), gate.data_ptr(), _lib.ptr(out_gate), _lib.ptr(slots), N,
                                      state.data_ptr(), out_state.data_ptr(), y.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "hyfft_gated_step")
    return y
