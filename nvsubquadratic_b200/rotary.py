"""Rotary positions of queries and keys.

Pair i of the first ``rot_dim`` features of every head is turned by ``position * frequency_i``. The frequencies
are laid out once, by ``rotary_turns``, as whole numbers (turns per position in units of 2^-64), so that whole turns drop out of
the 64-bit product exactly and far positions are as exact as near ones; the kernel (``hyfft_rotary`` in
``libhyfft.so``) computes the sines and cosines itself and reads no table. The reference's
rotary embedding lives in ``nvsubquadratic/utils/rope.py`` and serves its attention mixer.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

__all__ = ["rotary", "rotary_turns"]


def rotary_turns(rot_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_length: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0,
                 device=None) -> tuple[torch.Tensor, float]:
    """Frequencies for ``rot_dim`` turned features: ``(turns, amplitude)`` for ``rotary``.

    Pair i turns by ``base ** (-2 i / rot_dim)`` radians per position; ``scaling`` stretches that for contexts
    ``factor`` times longer than the ``original_length`` a model was trained on:

    * ``"none"``: as it is;
    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base multiplied by ``factor ** (rot_dim / (rot_dim - 2))``, which divides the slowest frequency by
      ``factor`` and leaves the fastest;
    * ``"ramp"``: pairs that turn more than ``fast_turns`` times within ``original_length`` keep their
      frequency, pairs that turn less than ``slow_turns`` times are divided by ``factor``, those between are blended by
      their index (from the whole number below the index that turns ``fast_turns`` times to the one above that of
      ``slow_turns``, which may lie past the last pair; at most ``rot_dim - 1``); the amplitude is ``0.1 ln(factor) + 1``.

    ``turns`` is int64 ``[rot_dim // 2]``, turns per position in units of 2^-64; ``amplitude`` is 1 but for ``"ramp"``.
    """
    assert rot_dim >= 2 and rot_dim % 2 == 0, f"rot_dim must be even and positive; got {rot_dim}"
    assert base > 1.0, f"base must be above 1; got {base}"
    assert factor >= 1.0, f"factor must be at least 1; got {factor}"
    half, amplitude = rot_dim // 2, 1.0
    if scaling == "ntk":
        base = base * factor ** (rot_dim / max(rot_dim - 2, 1))
    freq = [base ** (-2.0 * i / rot_dim) for i in range(half)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "ramp":
        assert original_length is not None and original_length > 0, 'scaling="ramp" needs original_length'

        def pair_turning(times):  # the index (a real number) of the pair that turns so often
            return rot_dim * math.log(original_length / (times * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_turning(fast_turns)), 0), min(math.ceil(pair_turning(slow_turns)), rot_dim - 1)
        for i in range(half):
            keep = 1.0 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            freq[i] = freq[i] / factor * (1.0 - keep) + freq[i] * keep
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}: use 'none', 'linear', 'ntk' or 'ramp'")
    turns = torch.tensor([int(f / (2 * math.pi) * 2.0 ** 64) for f in freq], dtype=torch.int64, device=device)
    return turns, amplitude


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_DESCS: dict = {}


def _desc(q, k, turns, positions, amplitude, interleaved, backward):
    """The descriptor of a call, built once for each set of shapes and strides."""
    key = (q.shape, q.stride(), q.dtype, None if k is None else (k.shape, k.stride()), turns.shape,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype), amplitude, interleaved,
           backward)
    d = _DESCS.get(key)
    if d is not None:
        return d
    d = _lib.RotaryDesc()
    d.batch, d.length, d.heads, d.dim = q.shape
    d.kv_heads = k.shape[2] if k is not None else 0
    d.rot_dim = 2 * turns.numel()
    d.dtype = _lib.DTYPE_CODE[q.dtype]
    d.interleaved, d.backward = int(interleaved), int(backward)
    d.amplitude = amplitude
    for i in range(3):
        d.q_stride[i] = q.stride(i)
        d.k_stride[i] = k.stride(i) if k is not None else 0
    if positions is not None:
        d.pos_int32 = int(positions.dtype == torch.int32)
        d.pos_stride[0] = positions.stride(0) if positions.ndim == 2 else 0
        d.pos_stride[1] = positions.stride(-1)
    if len(_DESCS) >= 256:
        _DESCS.clear()
    _DESCS[key] = d
    return d


def _call(q, k, turns, positions, amplitude, interleaved, backward):
    dev = _lib.require_cuda(q, k, turns, positions)
    q, k = _unit(q), _unit(k) if k is not None else None
    oq = q.new_empty(q.shape)
    ok = k.new_empty(k.shape) if k is not None else None
    if oq.numel() == 0:
        return oq, ok
    d = _desc(q, k, turns, positions, amplitude, interleaved, backward)
    rc = _lib.load().hyfft_rotary(ctypes.byref(d), q.data_ptr(), _lib.ptr(k), turns.data_ptr(), _lib.ptr(positions),
                                  oq.data_ptr(), _lib.ptr(ok), _lib.stream_ptr(dev))
    _lib.check(rc, "hyfft_rotary")
    return oq, ok


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, turns, positions, amplitude, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(turns, positions)
        ctx.args = (amplitude, interleaved)
        return _call(q, k, turns, positions, amplitude, interleaved, False)

    @staticmethod
    @_lib.no_second_derivative
    def backward(ctx, dq, dk):
        turns, positions = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 6
        if dq is None:  # one launch for what there is
            dk, _ = _call(dk, None, turns, positions, *ctx.args, True)
        else:
            dq, dk = _call(dq, dk, turns, positions, *ctx.args, True)
        return dq, dk, None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, turns: torch.Tensor, *, positions: torch.Tensor | None = None,
           amplitude: float = 1.0, interleaved: bool = False):
    """Turns queries and keys to their positions, both in one launch.

    Args:
        q ``[B, L, H, D]``, k ``[B, L, Hk, D]`` or None: float32, bfloat16 or float16, any batch, token and head strides.
        turns, amplitude: from ``rotary_turns``; ``2 * len(turns)`` features are turned, the others are copied.
        positions: int64 or int32, ``[L]`` or ``[B, L]``; ``0 .. L - 1`` by default.
        interleaved: pairs are neighbours ``(2i, 2i + 1)``; by default the two halves ``(i, i + rot_dim / 2)``.

    Returns ``(q', k')`` (k' None without k), contiguous, computed in float32 and rounded once. First derivatives only.
    """
    assert q.ndim == 4, f"q must be [B, L, H, D]; got {tuple(q.shape)}"
    B, L, H, D = q.shape
    assert H >= 1, "q must have a head"
    if k is not None:
        assert k.ndim == 4 and k.shape[:2] == q.shape[:2] and k.shape[3] == D and k.shape[2] >= 1, (
            f"k must be [{B}, {L}, heads, {D}]; got {tuple(k.shape)}")
        assert k.dtype == q.dtype, f"q and k must share a dtype; got {q.dtype} and {k.dtype}"
    assert turns.ndim == 1 and turns.dtype == torch.int64, "turns must be int64 [rot_dim // 2] (see rotary_turns)"
    assert 1 <= turns.numel() and 2 * turns.numel() <= D, (
        f"{2 * turns.numel()} features to turn do not fit heads of {D}")
    if positions is not None:
        assert positions.dtype in (torch.int64, torch.int32), f"positions must be int64 or int32; got {positions.dtype}"
        assert tuple(positions.shape) in ((L,), (B, L)), f"positions must be [{L}] or [{B}, {L}]; got {tuple(positions.shape)}"
    if q.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"dtype {q.dtype} is not supported (float32, bfloat16, float16)")
    args = (q, k, turns.contiguous(), positions, float(amplitude), bool(interleaved))
    if _lib.autograd_sees(q, k):
        return _RotaryFunction.apply(*args)
    return _call(*args, False)
