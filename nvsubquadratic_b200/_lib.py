"""ctypes binding of ``libhyfft.so`` (the C ABI declared in ``include/hyfft.h``).

This is the Python-side equivalent of the FFI a maintainer would add to
nvSubquadratic for the new backend. There is no CPU fallback: if the shared
library is missing or the tensors are not on a CUDA device, calls raise.
"""

from __future__ import annotations

import ctypes
import functools
import os
import threading
from pathlib import Path

import torch
from torch.autograd import forward_ad as _forward_ad

_PKG = Path(__file__).resolve().parent
_LIB_PATH = _PKG / "libhyfft.so"

HYFFT_OK = 0
HYFFT_ERR_INVALID = 1
HYFFT_ERR_UNSUPPORTED = 2
HYFFT_ERR_WORKSPACE = 3
HYFFT_ERR_CUDA = 4
HYFFT_ERR_WAIT = 5

F32, BF16, F16 = 0, 1, 2
LAYOUT_BHL, LAYOUT_BLH = 0, 1
GATE_IDENTITY, GATE_SIGMOID, GATE_SILU = 0, 1, 2

DTYPE_CODE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
GATE_CODE = {"identity": GATE_IDENTITY, "sigmoid": GATE_SIGMOID, "silu": GATE_SILU}


class ConvDesc(ctypes.Structure):
    _fields_ = [
        ("ndim", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("n", ctypes.c_int32 * 3),
        ("k", ctypes.c_int32 * 3),
        ("kernel_batch", ctypes.c_int32),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("layout", ctypes.c_int32),
        ("periodic", ctypes.c_int32),
    ]


class HyenaDesc(ctypes.Structure):
    _fields_ = [
        ("ndim", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("n", ctypes.c_int32 * 3),
        ("k", ctypes.c_int32 * 3),
        ("causal", ctypes.c_int32),
        ("short_k", ctypes.c_int32 * 3),
        ("short_causal", ctypes.c_int32),
        ("short_bias", ctypes.c_int32),
        ("gate1", ctypes.c_int32),
        ("gate2", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("in_batch_stride", ctypes.c_int64),
        ("in_pos_stride", ctypes.c_int64),
        ("out_batch_stride", ctypes.c_int64),
        ("out_pos_stride", ctypes.c_int64),
        ("periodic", ctypes.c_int32),
    ]


_vp = ctypes.c_void_p
_sz = ctypes.c_size_t
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32

# name -> argtypes (restype is int unless listed in _STR_FUNCS)
class SirenDesc(ctypes.Structure):
    _fields_ = [
        ("ndim", ctypes.c_int32),
        ("n", ctypes.c_int32 * 3),
        ("embedding", ctypes.c_int32),
        ("hidden", ctypes.c_int32),
        ("num_hidden", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("layout", ctypes.c_int32),
    ]


class DecayDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32),
        ("dk", ctypes.c_int32),
        ("dv", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("length", ctypes.c_int64),
        ("scale", ctypes.c_float),
        ("reserved", ctypes.c_int32),
        ("q_stride", ctypes.c_int64 * 3),
        ("k_stride", ctypes.c_int64 * 3),
        ("v_stride", ctypes.c_int64 * 3),
        ("o_stride", ctypes.c_int64 * 3),
    ]


class RotaryDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32),
        ("dim", ctypes.c_int32),
        ("rot_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("interleaved", ctypes.c_int32),
        ("backward", ctypes.c_int32),
        ("pos_int32", ctypes.c_int32),
        ("amplitude", ctypes.c_float),
        ("length", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 3),
        ("k_stride", ctypes.c_int64 * 3),
        ("pos_stride", ctypes.c_int64 * 2),
    ]


class GatedDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("form", ctypes.c_int32),
        ("complement", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("length", ctypes.c_int64),
        ("x_stride", ctypes.c_int64 * 2),
        ("gate_stride", ctypes.c_int64 * 2),
        ("out_gate_stride", ctypes.c_int64 * 2),
        ("dy_stride", ctypes.c_int64 * 2),
    ]


class QkNormDesc(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32),
        ("dim", ctypes.c_int32),
        ("rot_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("weight_dtype", ctypes.c_int32),
        ("interleaved", ctypes.c_int32),
        ("pos_int32", ctypes.c_int32),
        ("amplitude", ctypes.c_float),
        ("eps", ctypes.c_float),
        ("reserved", ctypes.c_int32),
        ("length", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 3),
        ("k_stride", ctypes.c_int64 * 3),
        ("dq_stride", ctypes.c_int64 * 3),
        ("dk_stride", ctypes.c_int64 * 3),
        ("pos_stride", ctypes.c_int64 * 2),
    ]


class Pool(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("row_bytes", ctypes.c_int64)]


SIGNATURES = {
    "hyfft_conv_workspace_size": [ctypes.POINTER(ConvDesc), ctypes.POINTER(_sz), ctypes.POINTER(_sz)],
    "hyfft_conv_forward": [ctypes.POINTER(ConvDesc), _vp, _vp, _vp, _vp, _vp, _sz, _vp],
    "hyfft_conv_forward_static_scratch": [ctypes.POINTER(ConvDesc), _vp, _vp, _vp, _vp, _vp],
    "hyfft_conv_backward": [ctypes.POINTER(ConvDesc), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp],
    "hyfft_hyena_workspace_size": [ctypes.POINTER(HyenaDesc), ctypes.POINTER(_sz), ctypes.POINTER(_sz),
                                   ctypes.POINTER(_sz)],
    "hyfft_hyena_forward": [ctypes.POINTER(HyenaDesc), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp],
    "hyfft_hyena_backward": [ctypes.POINTER(HyenaDesc), _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                             _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp],
    "hyfft_cp_pack_split_to_full": [_vp, _vp, _i64, _i64, _i64, _i64, _i32, _i32, _vp],
    "hyfft_cp_unpack_split_to_full": [_vp, _vp, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _vp],
    "hyfft_cp_pack_full_to_split": [_vp, _vp, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _vp],
    "hyfft_cp_unpack_full_to_split": [_vp, _vp, _i64, _i64, _i64, _i64, _i32, _i32, _vp],
    "hyfft_cp_permute_cl": [_vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _vp],
    "hyfft_cp_permute_cl_window": [_vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i32, _i64, _i64, _i32, _vp],
    "hyfft_causal_conv1d_forward": [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _vp],
    "hyfft_causal_conv1d_backward": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _vp],
    "hyfft_siren_sizes": [ctypes.POINTER(SirenDesc), ctypes.POINTER(_sz), ctypes.POINTER(_sz)],
    "hyfft_siren_forward": [ctypes.POINTER(SirenDesc)] + [_vp] * 10 + [_sz, _vp],
    "hyfft_siren_backward": [ctypes.POINTER(SirenDesc)] + [_vp] * 16 + [_sz, _vp],
    "hyfft_decay_workspace_size": [ctypes.POINTER(DecayDesc), ctypes.POINTER(_sz), ctypes.POINTER(_sz)],
    "hyfft_decay_saved_size": [ctypes.POINTER(DecayDesc), ctypes.POINTER(_sz)],
    "hyfft_decay_forward": [ctypes.POINTER(DecayDesc)] + [_vp] * 9 + [_sz, _vp],
    "hyfft_decay_backward": [ctypes.POINTER(DecayDesc)] + [_vp] * 15 + [_sz, _vp],
    "hyfft_decay_step": [ctypes.POINTER(DecayDesc)] + [_vp] * 5 + [_i64] + [_vp] * 4,
    "hyfft_rotary": [ctypes.POINTER(RotaryDesc)] + [_vp] * 7,
    "hyfft_layer_norm_workspace_size": [_i64, _i64, ctypes.POINTER(_sz)],
    "hyfft_layer_norm_forward": [_vp] * 6 + [_i64, _i64, _i64, ctypes.c_float, _i32, _i32, _vp],
    "hyfft_layer_norm_backward": [_vp] * 8 + [_i64, _i64, _i64, _i64, _i32, _i32, _vp, _sz, _vp],
    "hyfft_gated_saved_size": [ctypes.POINTER(GatedDesc), ctypes.POINTER(_sz)],
    "hyfft_gated_forward": [ctypes.POINTER(GatedDesc)] + [_vp] * 8 + [_sz, _vp],
    "hyfft_gated_backward": [ctypes.POINTER(GatedDesc)] + [_vp] * 5 + [_sz] + [_vp] * 7,
    "hyfft_gated_step": [ctypes.POINTER(GatedDesc)] + [_vp] * 4 + [_i64] + [_vp] * 4,
    "hyfft_qk_norm_workspace_size": [ctypes.POINTER(QkNormDesc), ctypes.POINTER(_sz)],
    "hyfft_qk_norm_forward": [ctypes.POINTER(QkNormDesc)] + [_vp] * 9,
    "hyfft_qk_norm_backward": [ctypes.POINTER(QkNormDesc)] + [_vp] * 13 + [_sz, _vp],
    "hyfft_pool_workspace_size": [_i64, _i64, ctypes.POINTER(_sz), ctypes.POINTER(_sz)],
    "hyfft_pool_copy": [ctypes.POINTER(Pool), _i32, _i64, _vp, _vp, _i64, _vp, _sz, _vp],
    "hyfft_pool_compact": [ctypes.POINTER(Pool), _i32, _i64, _vp, _vp, _vp, _sz, _vp],
    "hyfft_last_error": [],
    "hyfft_version": [],
    "hyfft_launch_count": [],
    "hyfft_wait_status": [_i32, _i32],
    "hyfft_set_wait_clocks": [ctypes.c_longlong],
}
_STR_FUNCS = {"hyfft_last_error", "hyfft_version"}

_lib = None
_lock = threading.Lock()


def library_path() -> Path:
    return Path(os.environ.get("HYFFT_LIBRARY", str(_LIB_PATH)))


def load() -> ctypes.CDLL:
    """Load libhyfft.so once; raise ImportError if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not path.exists():
            raise ImportError(
                f"{path} not found: build the CUDA backend first "
                "(python -m nvsubquadratic_b200.build). There is no CPU fallback."
            )
        lib = ctypes.CDLL(str(path))
        for name, args in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = ctypes.c_char_p if name in _STR_FUNCS else ctypes.c_int
        lib.hyfft_launch_count.restype = ctypes.c_longlong
        lib.hyfft_set_wait_clocks.restype = ctypes.c_longlong
        _lib = lib
        return lib


class HyfftError(RuntimeError):
    pass


def check(rc: int, what: str) -> None:
    if rc == HYFFT_OK:
        return
    msg = load().hyfft_last_error().decode(errors="replace")
    if rc == HYFFT_ERR_INVALID:
        raise AssertionError(f"{what}: {msg}")
    if rc == HYFFT_ERR_UNSUPPORTED:
        raise NotImplementedError(f"{what}: {msg}")
    raise HyfftError(f"{what} failed (status {rc}): {msg}")


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "the b200 FFT-conv backend runs on CUDA tensors only (got a tensor on "
                f"{t.device}); there is no CPU fallback"
            )
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    if dev is None:
        raise RuntimeError("no CUDA tensor given")
    return dev


# the current stream's handle without building a Stream object (2 us a call), where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def check_waits(device: torch.device | int = 0, clear: bool = True) -> None:
    """Waits for the device and raises ``HyfftError`` if a wait inside one of its kernels has run out since the last
    such check (the results of that call hold NaN)."""
    index = device if isinstance(device, int) else torch.device(device).index or 0
    check(load().hyfft_wait_status(index, int(clear)), "hyfft_wait_status")


def autograd_sees(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd has to see a call: an input requires a gradient, or carries a forward-mode tangent (which needs no
    requires_grad; a Function without a jvp refuses it)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if _forward_ad._current_level < 0:
        return False
    return any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Final(torch.autograd.Function):
    """Its tensors, which nothing can be differentiated through."""

    @staticmethod
    def forward(ctx, anchor, *tensors):
        return tuple(t.view_as(t) for t in tensors)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this operator's gradient has no second derivative")


def no_second_derivative(backward):
    """Decorates a Function's backward whose kernels record no graph: under ``create_graph=True`` differentiating its gradients
    again is an error. (``once_differentiable`` says so only where the upstream gradient requires a gradient itself; these
    gradients depend on saved inputs too.)"""

    @functools.wraps(backward)
    def wrapped(ctx, *upstream):
        if not torch.is_grad_enabled():
            return backward(ctx, *upstream)
        with torch.no_grad():
            grads = backward(ctx, *upstream)
        anchor = torch.empty(0, requires_grad=True)
        final = iter(_Final.apply(anchor, *(g for g in grads if g is not None)))
        return tuple(None if g is None else next(final) for g in grads)

    return wrapped


def launch_count() -> int:
    """Kernels launched through libhyfft.so by this process so far."""
    return int(load().hyfft_launch_count())
