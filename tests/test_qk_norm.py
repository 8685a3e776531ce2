"""Norms of heads with rotary positions: the oracle and refusals (CPU), the kernels against the float64 oracle (GPU).

Tolerances. In float32 a row's mean of squares is a sum of at most 256 terms, 16 in a lane and five steps across lanes (21 * 2^-24 of
it, half of that in its root), the root and three products 6 * 2^-24, the turn 16 * 2^-24: 64 * 2^-24 of a row for the outputs and, two such
sums in a row, 128 * 2^-24 of the upstream row times 1 / rms for the inputs' gradients. A weight's gradient is a float32 sum of n terms in some
order: (n + 128) * 2^-24 of the sum of their sizes. 16-bit results are rounded once more: 2^-8 (bfloat16), 2^-11 (float16).
"""

import math

import pytest
import torch

from nvsubquadratic_b200.qk_norm import qk_norm_rotary
from nvsubquadratic_b200.rotary import rotary, rotary_turns
from oracle.qk_norm import qk_norm_rotary as oracle
from tests.conftest import rel_l2

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TOL = {d: 64 * 2.0 ** -24 + h for d, h in HALF_STEP.items()}
DTYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])


def _radians(turns):
    return None if turns is None else turns.double().cpu() / 2.0 ** 64 * 2 * math.pi


def _check_dx(want, got, x, dy, w, dtype, eps=1e-6):
    size = (dy.double() * (1 if w is None else w.double().abs().max())).norm(dim=-1) / x.double().square().mean(-1).add(eps).sqrt()
    err = (want - got.double().cpu()).norm(dim=-1)
    floor = 2.0 ** -25 * x.shape[-1] ** 0.5 if dtype is F16 else 0.0
    assert (err <= (128 * 2.0 ** -24) * size + HALF_STEP[dtype] * want.norm(dim=-1) + floor).all()


def _check_dw(want, got, x, dy, dtype, turns, **kw):
    n = x.shape[0] * x.shape[1] * x.shape[2]
    h = x.double() / x.double().square().mean(-1, keepdim=True).add(1e-6).sqrt()
    # a turned pair's terms are at most the pair's length
    size = (dy.double().abs().amax(-1, keepdim=True) * 2 * kw.get("amplitude", 1.0) * h.abs()).sum((0, 1, 2))
    err = (want - got.double().cpu()).abs()
    assert (err <= (n + 128) * 2.0 ** -24 * size + HALF_STEP[got.dtype] * want.abs() + 2.0 ** -25).all()


# ---------------------------------------------------------------- CPU


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_gradients_are_autograds(interleaved):
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(2, 3, 2, 10, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.randn(10, generator=g, dtype=torch.float64)
    freq = torch.tensor([1.0, 0.3, 0.1], dtype=torch.float64)
    x.requires_grad_(), w.requires_grad_()
    n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    angle = torch.arange(3.0, dtype=torch.float64)[:, None] * freq
    c, s = angle.cos()[:, None] * 1.2, angle.sin()[:, None] * 1.2
    a, b = (n[..., 0:6:2], n[..., 1:6:2]) if interleaved else (n[..., :3], n[..., 3:6])
    a, b = a * c - b * s, a * s + b * c
    y = torch.cat((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1), n[..., 6:]), -1)
    want = torch.autograd.grad(y, [x, w], dy)
    got = oracle(x, w, freq, amplitude=1.2, interleaved=interleaved, dy=dy)
    assert torch.allclose(got[0], y) and torch.allclose(got[1], want[0]) and torch.allclose(got[2], want[1])


def test_refusals():
    t, _ = rotary_turns(8)
    q, k, w = torch.randn(2, 3, 4, 16), torch.randn(2, 3, 2, 16), torch.ones(16)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk_norm_rotary(q, k, w, w, t)
    with pytest.raises(AssertionError, match="q must be"):
        qk_norm_rotary(q[0], k)
    with pytest.raises(AssertionError, match="k must be"):
        qk_norm_rotary(q, k[:, :2])
    with pytest.raises(AssertionError, match="q and k must share"):
        qk_norm_rotary(q, k.half())
    with pytest.raises(AssertionError, match="k_weight without k"):
        qk_norm_rotary(q, None, w, w)
    with pytest.raises(AssertionError, match="q_weight must be"):
        qk_norm_rotary(q, k, w[:8])
    with pytest.raises(AssertionError, match="k_weight must be torch.float32 or"):
        qk_norm_rotary(q, k, w, w.double())
    with pytest.raises(AssertionError, match="q_weight and k_weight must share"):
        qk_norm_rotary(q.half(), k.half(), w, w.half())
    with pytest.raises(AssertionError, match="do not fit"):
        qk_norm_rotary(q[..., :6], k[..., :6], None, None, t)
    with pytest.raises(AssertionError, match="int64"):
        qk_norm_rotary(q, k, None, None, t.int())
    with pytest.raises(AssertionError, match="positions must be int64"):
        qk_norm_rotary(q, k, None, None, t, positions=torch.zeros(3))
    with pytest.raises(AssertionError, match=r"positions must be \[3\]"):
        qk_norm_rotary(q, k, None, None, t, positions=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(AssertionError, match="eps"):
        qk_norm_rotary(q, k, eps=-1.0)
    with pytest.raises(NotImplementedError, match="float64"):
        qk_norm_rotary(q.double(), k.double())


def test_library_refusals():
    """At the C entry, on the host, before anything is launched."""
    import ctypes

    from nvsubquadratic_b200 import _lib

    lib, p, size = _lib.load(), ctypes.c_void_p(16), ctypes.c_size_t()

    def desc(**kw):
        d = _lib.QkNormDesc()
        d.batch, d.length, d.heads, d.kv_heads, d.dim, d.rot_dim, d.dtype, d.weight_dtype = 2, 3, 4, 2, 16, 8, _lib.BF16, _lib.BF16
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    assert lib.hyfft_qk_norm_workspace_size(desc(), ctypes.byref(size)) == 0 and size.value > 0
    for bad in (dict(heads=0), dict(kv_heads=-1), dict(rot_dim=7), dict(rot_dim=18), dict(dtype=5), dict(weight_dtype=_lib.F16)):
        assert lib.hyfft_qk_norm_workspace_size(desc(**bad), ctypes.byref(size)) == _lib.HYFFT_ERR_INVALID, bad
    assert lib.hyfft_qk_norm_workspace_size(desc(dim=257), ctypes.byref(size)) == _lib.HYFFT_ERR_UNSUPPORTED
    assert lib.hyfft_qk_norm_forward(desc(), p, p, None, None, None, None, p, p, None) == _lib.HYFFT_ERR_INVALID  # no turns
    assert lib.hyfft_qk_norm_forward(desc(), p, None, None, None, p, None, p, p, None) == _lib.HYFFT_ERR_INVALID  # no k
    back = [p, p, None, None, p, None, p, p, p, p]
    assert lib.hyfft_qk_norm_backward(desc(), *back, p, None, p, 1 << 30, None) == _lib.HYFFT_ERR_INVALID  # no such weight
    back[2] = p
    assert lib.hyfft_qk_norm_backward(desc(), *back, p, None, p, 8, None) == _lib.HYFFT_ERR_WORKSPACE


# ---------------------------------------------------------------- GPU

# B, L, H, Hk, D, rot
SHAPES = [(1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 2, 2), (2, 5, 3, 1, 64, 64), (2, 17, 4, 4, 128, 64), (1, 9, 2, 2, 80, 50), (3, 7, 5, 5, 33, 32),
          (2, 4, 1, 1, 256, 256), (1, 300, 20, 3, 64, 16), (2, 3, 2, 2, 7, 6), (1, 6, 2, 1, 255, 100), (2, 3, 2, 1, 96, 0), (1, 4, 3, 3, 200, 128),
          (2, 5, 2, 2, 128, 18), (1, 3, 2, 1, 72, 70)]


def _case(B, L, H, Hk, D, rot, dtype, where, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, dq, dk = ((r(B, L, h, D) * s).to(dtype) for h, s in ((H, 2), (Hk, 2), (H, 1), (Hk, 1)))
    pos = None
    if where == "far":
        pos = torch.randint(-(1 << 30), 1 << 30, (B, 1), generator=g) + torch.arange(L)
    elif where == "shared":
        pos = torch.randint(0, 5000, (L,), generator=g).to(torch.int32)
    return q, k, dq, dk, 1 + 0.3 * r(D), 1 + 0.3 * r(D), pos


@gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("where,weights", [("order", None), ("far", "same"), ("shared", "f32")])
@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype, where, weights, interleaved):
    q, k, dq, dk, wq, wk, pos = _case(*shape, dtype, where)
    turns = rotary_turns(shape[5])[0] if shape[5] else None
    wd = dtype if weights == "same" else F32
    wq, wk = (None, None) if weights is None else (wq.to(wd), wk.to(wd))
    kw = dict(positions=pos, amplitude=1.25, interleaved=interleaved)
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (q, k, wq, wk)]
    out = qk_norm_rotary(*leaves, turns.cuda() if turns is not None else None, positions=pos.cuda() if pos is not None else None,
                         amplitude=1.25, interleaved=interleaved)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], [dq.cuda(), dk.cuda()])
    for i, (x, d, w) in enumerate(((q, dq, wq), (k, dk, wk))):
        y, dx, dw = oracle(x, w, _radians(turns), dy=d, **kw)
        assert out[i].dtype == dtype and out[i].is_contiguous() and rel_l2(y, out[i]) <= TOL[dtype]
        _check_dx(dx, grads[i], x, d * 1.25, w, dtype)
        if w is not None:
            assert grads[2 + i].dtype == wd
            _check_dw(dw, grads[2 + i], x, d, dtype, turns, amplitude=1.25)
    with torch.no_grad():
        again = qk_norm_rotary(*leaves, turns.cuda() if turns is not None else None,
                               positions=pos.cuda() if pos is not None else None, amplitude=1.25, interleaved=interleaved)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])


@gpu
@DTYPES
def test_many_rows(dtype):
    """More rows than the backward's CTAs take at once; the sums over rows come out the same every time."""
    q, k, dq, dk, wq, wk, _ = _case(2, 3000, 8, 2, 64, 64, dtype, "order")
    turns = rotary_turns(64)[0]
    leaves = [t.cuda().requires_grad_() for t in (q, k, wq.to(dtype), wk.to(dtype))]
    runs = []
    for _ in range(2):
        out = qk_norm_rotary(*leaves, turns.cuda())
        runs.append([*out, *torch.autograd.grad(out, leaves, [dq.cuda(), dk.cuda()])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    for i, (x, d, w) in enumerate(((q, dq, wq.to(dtype)), (k, dk, wk.to(dtype)))):
        y, dx, dw = oracle(x, w, _radians(turns), dy=d)
        assert rel_l2(y, runs[0][i]) <= TOL[dtype]
        _check_dx(dx, runs[0][2 + i], x, d, w, dtype)
        _check_dw(dw, runs[0][4 + i], x, d, dtype, turns)


@gpu
@DTYPES
def test_strides_alignment_and_missing_parts(dtype):
    B, L, H, D = 2, 6, 3, 64
    q, k, dq, dk, w, _, _ = _case(B, L, H, H, D, 32, dtype, "order")
    turns = rotary_turns(32)[0]
    w = w.to(dtype)
    wants = [oracle(x, w, _radians(turns), dy=d) for x, d in ((q, dq), (k, dk))]
    t, wc = turns.cuda(), w.cuda()
    packed = torch.cat((q.flatten(2), k.flatten(2)), -1).cuda()
    views = [packed[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(2)]
    heads = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (q, k)]
    odd = [torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in (q, k)]
    apart = [torch.stack((x, x), -1).flatten(-2).cuda()[..., ::2] for x in (q, k)]
    one = [q[:1].cuda().expand(B, L, H, D), k.cuda()]
    for form in (views, heads, odd, apart):
        leaves = [x.detach().requires_grad_() for x in form]
        out = qk_norm_rotary(*leaves, wc, wc, t)
        ups = [torch.nn.functional.pad(d, (1, 1)).cuda()[..., 1:-1] for d in (dq, dk)]
        grads = torch.autograd.grad(out, leaves, ups)
        for (y, dx, _), o, g, x, d in zip(wants, out, grads, (q, k), (dq, dk)):
            assert rel_l2(y, o) <= TOL[dtype]
            _check_dx(dx, g, x, d, w, dtype)
    shared = qk_norm_rotary(*one, wc, wc, t)
    assert torch.equal(shared[0][0], qk_norm_rotary(q.cuda(), None, wc, None, t)[0][0])
    a, b = qk_norm_rotary(views[0], None, wc, None, t)
    assert b is None and rel_l2(wants[0][0], a) <= TOL[dtype]
    # a gradient for k and its weight alone, and for one weight of two
    kd, wd = k.cuda().requires_grad_(), wc.clone().requires_grad_()
    gk, gw = torch.autograd.grad([qk_norm_rotary(q.cuda(), kd, wc, wd, t)[1]], [kd, wd], [dk.cuda()])
    _check_dx(wants[1][1], gk, k, dk, w, dtype)
    _check_dw(wants[1][2], gw, k, dk, dtype, turns)
    (gw,) = torch.autograd.grad(qk_norm_rotary(q.cuda(), k.cuda(), wd, None, t)[0], [wd], dq.cuda())
    _check_dw(wants[0][2], gw, q, dq, dtype, turns)
    empty = views[0][:, :0].detach().requires_grad_()
    out = qk_norm_rotary(empty, None, wd, None, t)[0]
    assert out.shape == (B, 0, H, D) and (torch.autograd.grad(out.sum(), [empty, wd])[1] == 0).all()


@gpu
def test_is_the_norm_and_then_the_turn():
    q, k, *_ = (t.cuda() if t is not None else None for t in _case(2, 9, 3, 2, 64, 64, F32, "order"))
    turns = rotary_turns(64, device="cuda")[0]
    a, b = qk_norm_rotary(q, k, None, None, turns)
    n = qk_norm_rotary(q, k)
    want = rotary(n[0], n[1], turns)
    assert rel_l2(want[0], a) <= 2 * TOL[F32] and rel_l2(want[1], b) <= 2 * TOL[F32]


@gpu
def test_gradients_are_the_slopes():
    q, k, dq, dk, wq, wk, pos = _case(2, 9, 3, 2, 40, 24, F32, "far")
    turns, g = rotary_turns(24)[0], torch.Generator().manual_seed(1)
    leaves = [t.cuda().requires_grad_() for t in (q, wq)]
    y, _ = qk_norm_rotary(leaves[0], k.cuda(), leaves[1], wk.cuda(), turns.cuda(), positions=pos.cuda())
    grads = torch.autograd.grad(y, leaves, dq.cuda())
    for i, grad in enumerate(grads):
        d, ends = torch.randn((q, wq)[i].shape, generator=g).double(), []
        for sign in (1, -1):
            args = [q.double(), wq.double()]
            args[i] = args[i] + sign * 1e-5 * d
            ends.append((oracle(*args, _radians(turns), positions=pos) * dq.double()).sum().item())
        slope = (ends[0] - ends[1]) / 2e-5
        assert abs(slope - (grad.double().cpu() * d).sum().item()) <= 1e-5 * grad.double().norm().item() * d.norm().item()


@gpu
@DTYPES
def test_rows_of_zeros_of_large_and_of_bad_values(dtype):
    """A row of zeros stays zero, features whose squares overflow are normed like others, and an infinity or a NaN stays in its row."""
    q, _, dq, _, w, _, _ = _case(1, 6, 4, 1, 64, 64, dtype, "order")
    w = w.to(dtype)
    turns = rotary_turns(64)[0]
    q[0, 1, 2] = 0
    big = 3.0e4 if dtype is F16 else 1.0e30
    q[0, 2, 1] *= big / 10
    q[0, 3, 0, 5] = float("inf")
    q[0, 4, 3, 7] = float("nan")
    leaf = q.cuda().requires_grad_()
    y, _ = qk_norm_rotary(leaf, None, w.cuda(), None, turns.cuda())
    (dx,) = torch.autograd.grad(y, [leaf], dq.cuda())
    want, wdx, _ = oracle(q, w, _radians(turns), dy=dq)
    ok = torch.ones(1, 6, 4, dtype=torch.bool)
    ok[0, 3, 0] = ok[0, 4, 3] = False
    y, dx = y.detach().cpu(), dx.cpu()
    assert torch.isfinite(y[ok]).all() and rel_l2(want[ok], y[ok]) <= TOL[dtype]
    assert (y[0, 1, 2] == 0).all() and rel_l2(want[0, 2, 1], y[0, 2, 1]) <= TOL[dtype]
    assert torch.isfinite(dx[ok]).all()
    ordinary = ok.clone()
    ordinary[0, 1, 2] = ordinary[0, 2, 1] = False
    _check_dx(wdx[ordinary], dx[ordinary], q[ordinary], dq[ordinary], w, dtype)
    assert y[0, 3, 0].isnan().any() and y[0, 4, 3].isnan().all()


@gpu
def test_no_eps_and_a_group_with_idle_lanes():
    """eps = 0: rows that a group of lanes does not have must not reach the weights' sums."""
    q, k, dq, dk, wq, wk, _ = _case(1, 3, 3, 1, 64, 64, F32, "order")
    leaves = [t.cuda().requires_grad_() for t in (q, k, wq, wk)]
    out = qk_norm_rotary(*leaves, eps=0.0)
    grads = torch.autograd.grad(out, leaves, [dq.cuda(), dk.cuda()])
    for i, (x, d, w) in enumerate(((q, dq, wq), (k, dk, wk))):
        y, dx, dw = oracle(x, w, eps=0.0, dy=d)
        assert rel_l2(y, out[i]) <= TOL[F32] and torch.isfinite(grads[2 + i]).all()
        _check_dx(dx, grads[i], x, d, w, F32)
        _check_dw(dw, grads[2 + i], x, d, F32, None)


@gpu
def test_second_and_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    q = torch.randn(2, 5, 3, 64, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(qk_norm_rotary(q, None)[0].square().sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    q = q.detach()
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward mode AD"):
            qk_norm_rotary(forward_ad.make_dual(q, torch.ones_like(q)), None)


@gpu
def test_streams_and_graphs():
    """Two calls at once on streams of their own, and a captured training step replayed on new inputs."""
    q, k, dq, dk, wq, wk, _ = (t.cuda() if t is not None else None for t in _case(2, 70, 4, 2, 64, 64, BF16, "order"))
    turns = rotary_turns(64, device="cuda")[0]
    wq, wk = wq.bfloat16(), wk.bfloat16()
    want = qk_norm_rotary(q, k, wq, wk, turns)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(qk_norm_rotary(q, k, wq, wk, turns))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for out in outs for o, w in zip(out, want))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]

    def step():
        return torch.autograd.grad(qk_norm_rotary(*leaves, turns), leaves, [dq, dk])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for leaf in leaves:
            leaf.add_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    kept = [g.clone() for g in got]
    assert all(torch.equal(a, b) for a, b in zip(kept, step()))


@gpu
@pytest.mark.parametrize("D", [64, 33, 256])
@pytest.mark.parametrize("size", [1e-13, 1e-20, 1e-30, 1e-36])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_small_rows_without_eps(dtype, size, D):
    """Features whose squares are below float32's range, eps = 0 or of their squares' size: normed like others."""
    q, k, dq, dk, wq, wk, _ = _case(2, 5, 3, 2, D, 0, dtype, "order")
    q, k = (q.float() * size).to(dtype), (k.float() * size).to(dtype)
    q[0, 1] = (q[0, 1].float() / size).to(dtype)  # among ordinary rows
    for eps in (0.0, size * size if size > 1e-19 else 0.0):
        leaves = [t.cuda().requires_grad_() for t in (q, k, wq, wk)]
        out = qk_norm_rotary(*leaves, eps=eps)
        grads = torch.autograd.grad(out, leaves, [dq.cuda(), dk.cuda()])
        for i, (x, d, w) in enumerate(((q, dq, wq), (k, dk, wk))):
            y, dx, _ = oracle(x, w, eps=torch.tensor(eps, dtype=F32).double().item(), dy=d)
            assert rel_l2(y, out[i]) <= TOL[dtype]
            _check_dx(dx, grads[i], x, d, w, dtype, eps=eps)
            assert torch.isfinite(grads[2 + i]).all()
    zeros = torch.zeros(1, 2, 1, D, device="cuda", dtype=dtype)
    assert (qk_norm_rotary(zeros, None, eps=1e-30)[0] == 0).all()


@gpu
def test_rows_from_large_to_small_in_one_call():
    """Every size of float32 that has all its digits, in rows that share warps; features of one row as far apart as they go."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 40, 6, 48, generator=g) * 10.0 ** torch.linspace(-37, 37, 240).view(1, 40, 6, 1)
    x[0, ::7, :, 1::2] *= 1e-3
    for eps in (0.0, 1e-30, 1e-6):
        y, _ = qk_norm_rotary(x.cuda(), None, eps=eps)
        want = oracle(x, eps=torch.tensor(eps, dtype=F32).double().item())
        assert ((want - y.double().cpu()).norm(dim=-1) <= TOL[F32] * want.norm(dim=-1) + 2.0 ** -126).all()
