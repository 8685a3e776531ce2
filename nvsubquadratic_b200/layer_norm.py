"""Layer norm over the last axis, forward and backward (``hyfft_layer_norm_forward`` / ``_backward`` in
``libhyfft.so``): the norm of the blocks around the mixers, and of their heads. The reference takes
``torch.nn.LayerNorm`` for its residual blocks (``nvsubquadratic/modules/residual_block.py``).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib

__all__ = ["layer_norm", "LayerNormB200"]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as ``[rows, C]`` with unit stride inside a row: a view where its rows have one stride, else a copy."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_size(rows: int, C: int) -> int:
    size = ctypes.c_size_t()
    _lib.check(_lib.load().hyfft_layer_norm_workspace_size(rows, C, ctypes.byref(size)),
               "hyfft_layer_norm_workspace_size")
    return size.value


def _param_code(x, weight, bias) -> int:
    p = weight if weight is not None else bias
    return _lib.DTYPE_CODE[p.dtype] if p is not None else _lib.F32


def _forward(x, weight, bias, eps, keep):
    """(y, x as rows, weight, statistics [2, rows]: means, then reciprocal deviations; None unless kept)."""
    dev = _lib.require_cuda(x, weight, bias)
    x2 = _rows(x)
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    rows, C = x2.shape
    y = x.new_empty(x.shape)
    stats = x.new_empty((2, rows), dtype=torch.float32) if keep else None
    if rows:
        mean = stats.data_ptr() if keep else None
        rc = _lib.load().hyfft_layer_norm_forward(
            x2.data_ptr(), _lib.ptr(w), _lib.ptr(b), y.data_ptr(), mean, mean + 4 * rows if keep else None, rows, C,
            x2.stride(0), eps, _lib.DTYPE_CODE[x.dtype], _param_code(x, w, b), _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_layer_norm_forward")
    return y, x2, w, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, x2, w, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, w, stats)
        ctx.shape = x.shape
        ctx.bias = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @_lib.no_second_derivative
    def backward(ctx, dy):
        x2, w, stats = ctx.saved_tensors
        dev = x2.device
        rows, C = x2.shape
        want = ctx.needs_input_grad
        dy2 = _rows(dy.to(x2.dtype))
        dx = x2.new_empty(ctx.shape) if want[0] else None
        dw = w.new_empty(C) if w is not None and want[1] else None
        db = x2.new_empty(C, dtype=ctx.bias) if ctx.bias is not None and want[2] else None
        if not rows:
            return dx, dw.zero_() if dw is not None else None, db.zero_() if db is not None else None, None
        lib = _lib.load()
        ws, need = None, 0
        if dw is not None or db is not None:
            need = _workspace_size(rows, C)
            ws = _lib.workspace(need, dev)
        code = _lib.DTYPE_CODE[w.dtype] if w is not None else (
            _lib.DTYPE_CODE[ctx.bias] if ctx.bias is not None else _lib.F32)
        mean = stats.data_ptr()
        rc = lib.hyfft_layer_norm_backward(x2.data_ptr(), _lib.ptr(w), mean, mean + 4 * rows,
                                           dy2.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), rows, C,
                                           x2.stride(0), dy2.stride(0), _lib.DTYPE_CODE[x2.dtype], code,
                                           _lib.ptr(ws), need, _lib.stream_ptr(dev))
        _lib.check(rc, "hyfft_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of ``x [..., C]`` (float32, bfloat16 or
    float16). weight and bias ``[C]``, each optional, both of x's dtype or both float32. Statistics and sums are float32;
    the output is rounded once to x's dtype, the parameters' gradients once to theirs. First derivatives only."""
    assert x.ndim >= 1 and x.shape[-1] >= 1, f"x must be [..., C]; got {tuple(x.shape)}"
    C = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            assert tuple(p.shape) == (C,), f"{name} must be [{C}]; got {tuple(p.shape)}"
            assert p.dtype in (x.dtype, torch.float32), f"{name} must be {x.dtype} or float32; got {p.dtype}"
    if weight is not None and bias is not None:
        assert weight.dtype == bias.dtype, f"weight and bias must share a dtype; got {weight.dtype} and {bias.dtype}"
    if x.dtype not in _lib.DTYPE_CODE:
        raise NotImplementedError(f"dtype {x.dtype} is not supported (float32, bfloat16, float16)")
    if _lib.autograd_sees(x, weight, bias):
        return _LayerNormFunction.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class LayerNormB200(torch.nn.Module):
    """``layer_norm`` with ``torch.nn.LayerNorm``'s parameters (one normalised axis)."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if elementwise_affine else None
        self.bias = (torch.nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))
                     if elementwise_affine and bias else None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)
