"""Rotary positions: frequencies (CPU), refusals (CPU), and the kernel against the float64 oracle (GPU).

Tolerances (relative L2): an element is two products and a sum with a sine and a cosine good to 4 units of 2^-24 and an angle
good to pi * 2^-24: 16 * 2^-24 in float32, and one rounding to nearest more in 16 bits, at most 2^-8 of an element in
bfloat16 (8 significant bits) and 2^-11 in float16 (11).
"""

import math

import pytest
import torch

from nvsubquadratic_b200.rotary import rotary, rotary_turns
from oracle.rotary import rotary as oracle
from tests.conftest import rel_l2

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 16 * 2.0 ** -24, BF16: 2.0 ** -8 + 1e-6, F16: 2.0 ** -11 + 1e-6}


def _radians(turns):
    return turns.double() / 2.0 ** 64 * 2 * math.pi


# ---------------------------------------------------------------- CPU


def test_turns():
    t, amp = rotary_turns(8, base=100.0)
    want = torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64)
    assert amp == 1.0 and torch.allclose(_radians(t), want, rtol=1e-14)
    assert torch.allclose(_radians(rotary_turns(8, base=100.0, scaling="linear", factor=4.0)[0]), want / 4, rtol=1e-14)
    ntk = _radians(rotary_turns(8, base=100.0, scaling="ntk", factor=4.0)[0])
    assert ntk[0].item() == pytest.approx(1.0) and ntk[-1].item() == pytest.approx(want[-1].item() / 4)
    plain = _radians(rotary_turns(64)[0])
    ramp, amp = rotary_turns(64, scaling="ramp", factor=8.0, original_length=4096)
    ratio = plain / _radians(ramp)
    assert ratio[0].item() == pytest.approx(1.0) and ratio[-1].item() == pytest.approx(8.0)
    assert (ratio[1:] >= ratio[:-1] - 1e-12).all() and amp == pytest.approx(1 + 0.1 * math.log(8))
    turned = plain * 4096 / (2 * math.pi)
    assert torch.allclose(ratio[turned > 40], torch.ones(1, dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(ratio[turned < 0.7], torch.full((1,), 8.0, dtype=torch.float64), rtol=1e-12)


def test_refusals():
    t, _ = rotary_turns(8)
    q, k = torch.randn(2, 3, 4, 16), torch.randn(2, 3, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary(q, k, t)
    with pytest.raises(AssertionError, match="q must be"):
        rotary(q[0], k, t)
    with pytest.raises(AssertionError, match="k must be"):
        rotary(q, k[:, :2], t)
    with pytest.raises(AssertionError, match="share a dtype"):
        rotary(q, k.half(), t)
    with pytest.raises(AssertionError, match="do not fit"):
        rotary(q[..., :6], k[..., :6], t)
    with pytest.raises(AssertionError, match="int64"):
        rotary(q, k, t.int())
    with pytest.raises(AssertionError, match="positions must be int64"):
        rotary(q, k, t, positions=torch.zeros(3))
    with pytest.raises(AssertionError, match=r"positions must be \[3\]"):
        rotary(q, k, t, positions=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(NotImplementedError, match="float64"):
        rotary(q.double(), k.double(), t)
    for bad in (0, 7):
        with pytest.raises(AssertionError, match="rot_dim"):
            rotary_turns(bad)
    with pytest.raises(ValueError, match="unknown scaling"):
        rotary_turns(8, scaling="other")
    with pytest.raises(AssertionError, match="original_length"):
        rotary_turns(8, scaling="ramp", factor=2.0)


# ---------------------------------------------------------------- GPU

# B, L, H, Hk, D, rot
SHAPES = [(1, 1, 1, 1, 2, 2), (2, 5, 3, 1, 64, 64), (2, 17, 4, 4, 128, 64), (1, 9, 2, 2, 80, 50), (3, 7, 5, 5, 33, 32),
          (2, 4, 1, 1, 256, 256), (1, 300, 20, 3, 64, 16), (2, 3, 2, 2, 7, 6)]


def _case(B, L, H, Hk, D, rot, dtype, where, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(B, L, H, D, generator=g).to(dtype), torch.randn(B, L, Hk, D, generator=g).to(dtype)
    dq, dk = torch.randn(B, L, H, D, generator=g).to(dtype), torch.randn(B, L, Hk, D, generator=g).to(dtype)
    pos = None
    if where == "far":  # one start for each row, forwards and back, up to 2^30
        pos = torch.randint(-(1 << 30), 1 << 30, (B, 1), generator=g) + torch.arange(L)
    elif where == "shared":
        pos = torch.randint(0, 5000, (L,), generator=g).to(torch.int32)
    return q, k, dq, dk, pos


@gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("where", ["order", "far", "shared"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradient(shape, dtype, where, interleaved):
    q, k, dq, dk, pos = _case(*shape, dtype, where)
    turns, _ = rotary_turns(shape[5])
    freq, amp = _radians(turns), 1.25
    # the oracle's angle in float64 is good to 2^30 * 2^-53 radians
    kw = dict(positions=pos, amplitude=amp, interleaved=interleaved)
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = rotary(qd, kd, turns.cuda(), positions=pos.cuda() if pos is not None else None, amplitude=amp,
                 interleaved=interleaved)
    grads = torch.autograd.grad(out, [qd, kd], [dq.cuda(), dk.cuda()])
    for x, got in ((q, out[0]), (k, out[1])):
        assert got.dtype == dtype and rel_l2(oracle(x, freq, **kw), got) <= TOL[dtype]
    for d, got in ((dq, grads[0]), (dk, grads[1])):
        assert rel_l2(oracle(d, freq, backward=True, **kw), got) <= TOL[dtype]
    assert torch.equal(out[0].detach().cpu()[..., shape[5]:], q[..., shape[5]:])  # what is not turned is copied


@gpu
def test_gradient_is_the_slope():
    """The map is linear: <dy, f(x + d)> - <dy, f(x)> is <f^T dy, d> up to rounding."""
    q, k, dq, dk, pos = (t.cuda() for t in _case(2, 9, 3, 2, 40, 24, F32, "far"))
    turns = rotary_turns(24, device="cuda")[0]
    q.requires_grad_()
    y, _ = rotary(q, k, turns, positions=pos)
    (g,) = torch.autograd.grad(y, [q], dq)
    d = torch.randn_like(q)
    slope = ((rotary(q + d, k, turns, positions=pos)[0].double() - y.double()) * dq.double()).sum()
    assert abs(slope - (g.double() * d.double()).sum()) <= 4 * TOL[F32] * y.double().norm() * dq.double().norm()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides_alignment_and_missing_k(dtype):
    B, L, H, D = 2, 6, 3, 64
    q, k, dq, dk, _ = _case(B, L, H, H, D, 32, dtype, "order")
    turns = rotary_turns(32)[0]
    wq, wk = (oracle(t, _radians(turns)) for t in (q, k))
    t = turns.cuda()
    packed = torch.cat((q.flatten(2), k.flatten(2)), -1).cuda()
    views = [packed[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(2)]
    heads = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (q, k)]
    odd = [torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in (q, k)]
    apart = [torch.stack((x, x), -1).flatten(-2).cuda()[..., ::2] for x in (q, k)]
    for form in (views, heads, odd, apart):
        a, b = rotary(*form, t)
        assert a.is_contiguous() and rel_l2(wq, a) <= TOL[dtype] and rel_l2(wk, b) <= TOL[dtype]
    a, b = rotary(views[0], None, t)
    assert b is None and rel_l2(wq, a) <= TOL[dtype]
    kd = k.cuda().requires_grad_()  # a gradient for k alone
    out = rotary(q.cuda(), kd, t)
    (g,) = torch.autograd.grad([out[1]], [kd], [dk.cuda()])
    assert rel_l2(oracle(dk, _radians(turns), backward=True), g) <= TOL[dtype]
    assert rotary(views[0][:, :0], views[1][:, :0], t)[0].shape == (B, 0, H, D)


@pytest.mark.parametrize("rot,length", [(64, 131072), (64, 1 << 20), (128, 131072), (6, 8192), (8, 8192), (64, 4096), (32, 512)])
def test_ramp_follows_its_definition(rot, length):
    """Slowed by 8 below one turn within the original length, not at all above 32, in between by the index: 0 at the whole index below
    that of 32 turns, 1 at the one above that of one turn, wherever the last pair lies."""
    ratio = _radians(rotary_turns(rot)[0]) / _radians(rotary_turns(rot, scaling="ramp", factor=8.0, original_length=length)[0])
    # turns of a pair of index x: length * 10000^(-2 x / rot) / (2 pi)
    index = lambda turns: rot / 2 * (math.log(length / (2 * math.pi)) - math.log(turns)) / math.log(10000.0)  # noqa: E731
    low, high = max(math.floor(index(32.0)), 0), math.ceil(index(1.0))
    for i in range(rot // 2):
        slowed = min(max((i - low) / (high - low), 0.0), 1.0)
        assert ratio[i].item() == pytest.approx(1.0 / (1.0 - slowed + slowed / 8.0), rel=1e-12), i
        turns = length * 10000.0 ** (-2 * i / rot) / (2 * math.pi)
        if 1.0 < turns < 32.0 and low < i < high:
            assert 1.0 < ratio[i].item() < 8.0


@pytest.mark.parametrize("rot,length,last", [(64, 131072, 2.54), (64, 1 << 20, 1.16)])
def test_ramp_blends_a_last_pair_that_still_turns(rot, length, last):
    """Worked out by hand: the last pair (31) of 64 features turns 2.78 and 22 times; it is divided by less than the factor."""
    plain, ramp = (_radians(rotary_turns(rot, **a)[0]) for a in ({}, dict(scaling="ramp", factor=8.0, original_length=length)))
    assert (plain[-1] / ramp[-1]).item() == pytest.approx(last, abs=0.01)


@gpu
def test_second_and_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    q, k, dq, dk, _ = (t.cuda() if t is not None else None for t in _case(2, 5, 3, 1, 64, 64, F32, "order"))
    turns = rotary_turns(64, device="cuda")[0]
    q.requires_grad_()
    (g,) = torch.autograd.grad(rotary(q, k, turns)[0].square().sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (q.sum() + g.sum()).backward()
    q = q.detach()
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(q, dq), k), (q, forward_ad.make_dual(k, dk))):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward mode AD"):
                rotary(*args, turns)
