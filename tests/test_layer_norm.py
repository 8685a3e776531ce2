"""Layer norm: the oracle against differences and refusals (CPU), the kernels against the float64 oracle (GPU).

Tolerances (relative L2): float32 sums of C terms held by up to 512 threads add at most 32 rounded terms in one thread, then
trees: 64 * 2^-24 for outputs and gradients of inputs; the parameters' sums run over thousands of rows, independent
roundings: 128 * 2^-24. A 16-bit result is rounded once more, to nearest: at most 2^-8 of an element in bfloat16 (8
significant bits), 2^-11 in float16 (11).
"""

import pytest
import torch

from nvsubquadratic_b200.layer_norm import LayerNormB200, layer_norm
from oracle.layer_norm import layer_norm as oracle
from tests.conftest import rel_l2

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _tol(dtype, terms=64):
    return UNIT[dtype] + terms * 2.0 ** -24


# ---------------------------------------------------------------- CPU


def test_oracle_gradients_are_differences():
    torch.manual_seed(0)
    x, w, b, dy = (torch.randn(s, dtype=torch.float64) for s in ((5, 7), (7,), (7,), (5, 7)))
    grads = oracle(x, w, b, dy=dy)[1:]
    eps, args = 1e-5, [x, w, b]
    for i in range(3):
        d = torch.randn_like(args[i])
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * d, args[i] - eps * d
        slope = ((oracle(*up) - oracle(*down)) * dy).sum() / (2 * eps)
        assert slope.item() == pytest.approx((grads[i] * d).sum().item(), rel=1e-6, abs=1e-8)


def test_refusals():
    x = torch.randn(3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(AssertionError, match="weight must be"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(AssertionError, match="weight must be torch.bfloat16 or float32"):
        layer_norm(x.bfloat16(), torch.ones(8).half())
    with pytest.raises(AssertionError, match="share a dtype"):
        layer_norm(x.bfloat16(), torch.ones(8), torch.ones(8).bfloat16())
    with pytest.raises(NotImplementedError, match="float64"):
        layer_norm(x.double())


def test_module_parameters():
    m, ref = LayerNormB200(12), torch.nn.LayerNorm(12)
    assert {n: p.shape for n, p in m.state_dict().items()} == {n: p.shape for n, p in ref.state_dict().items()}
    assert LayerNormB200(12, bias=False).bias is None and not LayerNormB200(12, elementwise_affine=False).state_dict()


# ---------------------------------------------------------------- GPU

# rows, C
SHAPES = [(1, 1), (3, 2), (5, 31), (33, 64), (700, 96), (9, 255), (17, 256), (40, 257), (1300, 768), (3, 771), (2, 1024),
          (700, 4096), (3, 4097), (2, 8200), (3, 16384), (2, 16390), (2, 20001)]


def _case(rows, C, dtype, pdtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(rows, C, generator=g) + 0.7).to(dtype)
    dy = torch.randn(rows, C, generator=g).to(dtype)
    w, b = ((1 + 0.3 * torch.randn(C, generator=g)).to(pdtype), (0.2 * torch.randn(C, generator=g)).to(pdtype))
    return x, w, b, dy


@gpu
@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none", "float32"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype, affine):
    pdtype = F32 if affine == "float32" else dtype
    x, w, b, dy = _case(*shape, dtype, pdtype)
    if affine in ("bias", "none"):
        w = None
    if affine in ("weight", "none"):
        b = None
    want = oracle(x, w, b, dy=dy)
    args = [t.cuda().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = layer_norm(*args)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, [t for t in args if t is not None], dy.cuda())
    scale = 1.0 if shape[1] > 2 else 2.0 ** 10  # rows of one or two values: the oracle's own differences cancel
    assert rel_l2(want[0], y) <= _tol(dtype) * scale
    dx = grads[0].double().cpu()
    # dx of a short row is a difference of terms of dy's size: measured against those
    size = (dy.double() if w is None else dy.double() * w.double()).norm() / x.double().std().clamp(min=0.1)
    assert (dx - want[1]).norm() <= _tol(dtype) * max(want[1].norm(), scale * size if shape[1] <= 2 else 0)
    names = [n for n, t in zip(("dw", "db"), (w, b)) if t is not None]
    for n, got in zip(names, grads[1:]):
        assert got.dtype == pdtype
        assert rel_l2(want[2 if n == "dw" else 3], got) <= _tol(pdtype, 128) * (scale if n == "dw" else 1), n


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_far_from_zero_and_constant_rows(dtype):
    """A mean 1000 deviations away costs the mean's rounding only (no E[x^2] - E[x]^2); constant rows give the bias."""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-2, 3, (50, 512), generator=g).to(dtype)
    x = (x + 1000 if dtype is F32 else x + 100).to(dtype)  # whole numbers: exact in either type
    w, b = torch.ones(512, dtype=dtype), torch.full((512,), 0.5, dtype=dtype)
    assert rel_l2(oracle(x, w, b), layer_norm(x.cuda(), w.cuda(), b.cuda())) <= _tol(dtype, 1024)
    flat = torch.full((4, 512), 3.0, dtype=dtype).cuda()
    assert torch.equal(layer_norm(flat, w.cuda(), b.cuda()), torch.full_like(flat, 0.5))


@gpu
def test_bad_values_stay_in_their_row():
    x, w, b, dy = (t.cuda() for t in _case(6, 300, F32, F32))
    want = layer_norm(x, w, b)
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    got = layer_norm(x, w, b)
    keep = torch.tensor([0, 1, 3, 5])
    assert torch.equal(got[keep], want[keep]) and got[2].isnan().all() and got[4].isnan().any()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides_shapes_and_alignment(dtype):
    x, w, b, dy = _case(2 * 5 * 3, 64, dtype, dtype)
    x4, dy4 = x.view(2, 5, 3, 64), dy.view(2, 5, 3, 64)
    want = oracle(x4, w, b, dy=dy4)
    wide = torch.zeros(2, 5, 3, 100, dtype=dtype)
    wide[..., 3:67] = x4
    forms = [x4.cuda(), wide.cuda()[..., 3:67], x4.transpose(1, 2).contiguous().cuda().transpose(1, 2),
             torch.stack((x4, x4), -1).cuda()[..., 0]]
    for xf in forms:
        xf = xf.requires_grad_()
        wd, bd = w.cuda().requires_grad_(), b.cuda().requires_grad_()
        y = layer_norm(xf, wd, bd)
        up = torch.stack((dy4, dy4), 0).cuda()[1]
        dx, dw, db = torch.autograd.grad(y, [xf, wd, bd], up)
        assert y.shape == x4.shape and rel_l2(want[0], y) <= _tol(dtype) and rel_l2(want[1], dx) <= _tol(dtype)
        assert rel_l2(want[2], dw) <= _tol(dtype, 128) and rel_l2(want[3], db) <= _tol(dtype, 128)
    one = layer_norm(x[0].cuda(), w.cuda(), b.cuda())
    assert one.shape == (64,) and rel_l2(oracle(x[0], w, b), one) <= _tol(dtype)


@gpu
def test_no_rows_and_partial_gradients():
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 16, device="cuda"))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    x, w, b, dy = (t.cuda() for t in _case(100, 48, F32, F32))
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for i in range(3):
        part = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(layer_norm(*part), [part[i]], dy)
        assert torch.equal(got, want[i])
    assert not layer_norm(x, w, b).requires_grad


@gpu
def test_same_bits_every_time():
    x, w, b, dy = (t.cuda().requires_grad_() for t in _case(3000, 768, BF16, BF16))
    runs = [torch.autograd.grad(layer_norm(x, w, b), [x, w, b], dy) for _ in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*runs))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5000, 64), (3000, 768), (4000, 4096), (40, 8192)], ids=str)
def test_waits_that_run_out_leave_nan_and_a_status(shape, dtype):
    """With no patience at all the waits for rows run out: every value is the right one or NaN, the host can tell, and the
    next call is as ever."""
    from nvsubquadratic_b200 import _lib

    x, w, b, dy = (t.cuda() for t in _case(*shape, dtype, dtype))
    args = [t.requires_grad_() for t in (x, w, b)]

    def run():
        y = layer_norm(*args)
        return [y.detach(), *torch.autograd.grad(y, args, dy)]

    want = run()
    _lib.check_waits(0)
    lib = _lib.load()
    before = lib.hyfft_set_wait_clocks(0)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        lib.hyfft_set_wait_clocks(before)
    # a row may have arrived before it is asked for: there is a status exactly where there is a NaN
    if any(t.isnan().any() for t in got):
        with pytest.raises(_lib.HyfftError, match="layer norm"):
            _lib.check_waits(0)
    else:
        assert shape[1] < 4096  # groups that walk over many wide rows do not find every one there
    _lib.check_waits(0)
    for p, q in zip(want, got):
        assert ((p == q) | q.isnan()).all()
    assert all(torch.equal(p, q) for p, q in zip(want, run()))
    _lib.check_waits(0)


# ---------------------------------------------------------------- derivatives that are not there


def test_autograd_sees_tangents():
    from torch.autograd import forward_ad

    from nvsubquadratic_b200 import _lib

    plain, leaf = torch.randn(3), torch.randn(3, requires_grad=True)
    assert _lib.autograd_sees(None, leaf) and not _lib.autograd_sees(plain, None)
    with torch.no_grad():
        assert not _lib.autograd_sees(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(plain, torch.ones(3))
        assert _lib.autograd_sees(None, dual) and not _lib.autograd_sees(plain)
        with torch.no_grad():
            assert _lib.autograd_sees(dual)
    assert not _lib.autograd_sees(plain)


@gpu
def test_second_and_forward_mode_derivatives_are_refused():
    """Neither has a kernel: an error, not a result that lacks them."""
    from torch.autograd import forward_ad

    x, w, b, dy = (t.cuda() for t in _case(5, 64, F32, F32))
    x.requires_grad_()
    (dx,) = torch.autograd.grad(layer_norm(x, w, b), [x], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):  # a penalty beside a loss
        (x.sum() + dx.square().sum()).backward()
    x = x.detach()
    for i in range(3):
        with forward_ad.dual_level():
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((x, w, b))]
            with pytest.raises((RuntimeError, NotImplementedError), match="forward mode AD"):
                layer_norm(*args)
            layer_norm(x, w, b)  # nothing to lose


def test_gradients_without_a_second_derivative():
    from nvsubquadratic_b200 import _lib

    class Square(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y):
            ctx.save_for_backward(x)
            return x.square() + y

        @staticmethod
        @_lib.no_second_derivative
        def backward(ctx, g):
            return 2 * g * ctx.saved_tensors[0], None

    x = torch.randn(3, requires_grad=True)
    (g,) = torch.autograd.grad(Square.apply(x, torch.zeros(3)).sum(), [x])
    assert not g.requires_grad and torch.equal(g, 2 * x.detach())
    (g,) = torch.autograd.grad(Square.apply(x, torch.zeros(3)).sum(), [x], create_graph=True)
    assert torch.equal(g.detach(), 2 * x.detach())
    with pytest.raises(RuntimeError, match="second derivative"):
        (x.sum() + g.sum()).backward()
