"""The norm of every head of queries and keys, with rotary positions in the same pass.

Each head of each token is divided by its root mean square and scaled by a weight for each feature, then its pairs are turned to
their positions as by ``rotary``: one read of q and k and one write, where a norm and a rotation apart take two of each. The
computation runs in ``libhyfft.so`` (``hyfft_qk_norm_forward`` / ``_backward``), with no CPU fallback. The reference
normalises queries and keys by their length (``nvsubquadratic/utils/qk_norm.py``) and turns them in ``nvsubquadratic/utils/rope.py``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["qk_norm_rotary"]


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_DESCS: dict = {}


def _desc(q, k, q_weight, k_weight, turns, positions, eps, amplitude, interleaved, dq=None, dk=None):
    """(descriptor, bytes of the backward's workspace) of a call, built once for each set of shapes and strides."""
    weight = q_weight if q_weight is not None else k_weight
    key = (q.shape, q.stride(), q.dtype, None if k is None else (k.shape, k.stride()), None if weight is None else weight.dtype,
           None if turns is None else turns.shape,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype), eps, amplitude, interleaved,
           None if dq is None else dq.stride(), None if dk is None else dk.stride())
    hit = _DESCS.get(key)
    if hit is not None:
        return hit
    d = _lib.QkNormDesc()
    d.batch, d.length, d.heads, d.dim = q.shape
    d.kv_heads = k.shape[2] if k is not None else 0
    d.rot_dim = 2 * turns.numel() if turns is not None else 0
    d.dtype = _lib.DTYPE_CODE[q.dtype]
    d.weight_dtype = _lib.DTYPE_CODE[weight.dtype] if weight is not None else d.dtype
    d.interleaved, d.eps, d.amplitude = int(interleaved), eps, amplitude
    for to, t in ((d.q_stride, q), (d.k_stride, k), (d.dq_stride, dq), (d.dk_stride, dk)):
        if t is not None:  # the stride of an axis of one entry is not used, and may be anything
            for i in range(3):
                to[i] = t.stride(i) if t.shape[i] > 1 else 0
    if positions is not None:
        d.pos_int32 = int(positions.dtype == torch.int32)
        d.pos_stride[0] = positions.stride(0) if positions.ndim == 2 else 0
        d.pos_stride[1] = positions.stride(-1)
    size = ctypes.c_size_t()
    _lib.check(_lib.load().hyfft_qk_norm_workspace_size(ctypes.byref(d), ctypes.byref(size)), "hyfft_qk_norm_workspace_size")
    if len(_DESCS) >= 256:
        _DESCS.clear()
    _DESCS[key] = hit = (d, size.value)
    return hit


def _forward(q, k, q_weight, k_weight, turns, positions, *args):
    dev = _lib.require_cuda(q, k, q_weight, k_weight, turns, positions)
    q, k = _unit(q), _unit(k) if k is not None else None
    oq = q.new_empty(q.shape)
    ok = k.new_empty(k.shape) if k is not None else None
    if oq.numel():
        d, _ = _desc(q, k, q_weight, k_weight, turns, positions, *args)
        rc = _lib.load().hyfft_qk_norm_forward(ctypes.byref(d), q.data_ptr(), _lib.ptr(k), _lib.ptr(q_weight),
                                               _lib.ptr(k_weight), _lib.ptr(turns), _lib.ptr(positions), oq.data_ptr(),
                                               _lib.ptr(ok), _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_qk_norm_forward")
    return oq, ok


class _QkNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, turns, positions, *args):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, turns, positions)
        ctx.args = args
        return _forward(q, k, q_weight, k_weight, turns, positions, *args)

    @staticmethod
    @_lib.no_second_derivative
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, turns, positions = ctx.saved_tensors
        none = (None,) * 5
        if dq is None and dk is None:
            return (None,) * 4 + none
        if dq is None:  # one launch for what there is
            gk, _, wk, _ = _backward(k, None, k_weight, None, turns, positions, ctx.args, dk, None, ctx.needs_input_grad[3], False)
            return None, gk, None, wk, *none
        if dk is None:
            gq, _, wq, _ = _backward(q, None, q_weight, None, turns, positions, ctx.args, dq, None, ctx.needs_input_grad[2], False)
            return gq, None, wq, None, *none
        return *_backward(q, k, q_weight, k_weight, turns, positions, ctx.args, dq, dk, *ctx.needs_input_grad[2:4]), *none


def _backward(q, k, q_weight, k_weight, turns, positions, args, dq, dk, want_qw, want_kw):
    q, dq = _unit(q), _unit(dq.to(q.dtype))
    k, dk = (_unit(k), _unit(dk.to(k.dtype))) if k is not None else (None, None)
    gq = q.new_empty(q.shape)
    gk = k.new_empty(k.shape) if k is not None else None
    wq = torch.empty_like(q_weight) if want_qw else None
    wk = torch.empty_like(k_weight) if want_kw else None
    if not gq.numel():
        return gq, gk, wq.zero_() if wq is not None else None, wk.zero_() if wk is not None else None
    d, size = _desc(q, k, q_weight, k_weight, turns, positions, *args, dq, dk)
    ws = _lib.workspace(size, q.device) if want_qw or want_kw else None
    rc = _lib.load().hyfft_qk_norm_backward(ctypes.byref(d), q.data_ptr(), _lib.ptr(k), _lib.ptr(q_weight), _lib.ptr(k_weight),
                                            _lib.ptr(turns), _lib.ptr(positions), dq.data_ptr(), _lib.ptr(dk), gq.data_ptr(),
                                            _lib.ptr(gk), _lib.ptr(wq), _lib.ptr(wk), _lib.ptr(ws), size,
                                            _lib.stream_ptr(q.device))
    _lib.check(rc, "hyfft_qk_norm_backward")
    return gq, gk, wq, wk


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, turns: torch.Tensor | None = None, *, eps: float = 1e-6,
                   positions: torch.Tensor | None = None, amplitude: float = 1.0, interleaved: bool = False):
    """``x / sqrt(mean(x ** 2) + eps) * weight`` over the features of each head, then turned to its position; queries and keys in
    one launch.

    Args:
        q ``[B, L, H, D]``, k ``[B, L, Hk, D]`` or None: float32, bfloat16 or float16, any batch, token and head strides. D <= 256.
        q_weight, k_weight: ``[D]`` each, shared by the heads, both of q's dtype or both float32; None: 1.
        turns, amplitude: from ``rotary_turns``; ``2 * len(turns)`` features are turned, the others are normed alone. None: no turn.
        eps: 0 or more; with 0 a row of zeros is NaN, and one whose features are all below 2^-126 is not normed.
        positions: int64 or int32, ``[L]`` or ``[B, L]``; ``0 .. L - 1`` by default.
        interleaved: pairs are neighbours ``(2i, 2i + 1)``; by default the two halves ``(i, i + rot_dim / 2)``.

    Returns ``(q', k')`` (k' None without k), contiguous. Computed in float32 and rounded once, the weights' gradients too. First
    derivatives only.
    """
    assert q.ndim == 4, f"q must be [B, L, H, D]; got {tuple(q.shape)}"
    B, L, H, D = q.shape
    assert H >= 1 and D >= 1, "q must have a head and features"
    if k is not None:
        assert k.ndim == 4 and k.shape[:2] == q.shape[:2] and k.shape[3] == D and k.shape[2] >= 1, (
            f"k must be [{B}, {L}, heads, {D}]; got {tuple(k.shape)}")
        assert k.dtype == q.dtype, f"q and k must share a dtype; got {q.dtype} and {k.dtype}"
    assert k is not None or k_weight is None, "k_weight without k"
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            assert tuple(w.shape) == (D,), f"{name} must be [{D}]; got {tuple(w.shape)}"
            assert w.dtype in (q.dtype, torch.float32), f"{name} must be {q.dtype} or float32; got {w.dtype}"
    if q_weight is not None and k_weight is not None:
        assert q_weight.dtype == k_weight.dtype, (
            f"q_weight and k_weight must share a dtype; got {q_weight.dtype} and {k_weight.dtype}")
    if turns is not None:
        assert turns.ndim == 1 and turns.dtype == torch.int64, "turns must be int64 [rot_dim // 2] (see rotary_turns)"
        assert 1 <= turns.numel() and 2 * turns.numel() <= D, (
            f"{2 * turns.numel()} features to turn do not fit heads of {D}")
    if positions is not None:
        assert positions.dtype in (torch.int64, torch.int32), f"positions must be int64 or int32; got {positions.dtype}"
        assert tuple(positions.shape) in ((L,), (B, L)), f"positions must be [{L}] or [{B}, {L}]; got {tuple(positions.shape)}"
    assert eps >= 0, f"eps must not be negative; got {eps}"
    if q.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"dtype {q.dtype} is not supported (float32, bfloat16, float16)")
    args = (q, k, q_weight.contiguous() if q_weight is not None else None, k_weight.contiguous() if k_weight is not None else None,
            turns.contiguous() if turns is not None else None, positions, float(eps), float(amplitude), bool(interleaved))
    if _lib.autograd_sees(q, k, q_weight, k_weight):
        return _QkNormFunction.apply(*args)
    return _forward(*args)
