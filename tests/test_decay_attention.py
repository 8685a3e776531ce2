"""Decayed linear attention: the float64 oracle against differences (CPU), refusals (CPU), and the kernels against the
oracle at the sizes, lengths, decays and strides where they can go wrong (GPU).

Tolerances (relative L2 over a tensor). A float32 result adds up to ~2^14 rounded terms whose errors are independent:
sqrt(2^14) * 2^-24 = 7.6e-6. A 16-bit result is rounded to nearest once, at most u of an element (u = 2^-8 in bfloat16, 2^-11
in float16, the rounding's RMS below u / sqrt(3)), and one operand of each of two products may be rounded to the
same type on the way: three independent errors of u / sqrt(3) are u, and half as much again is allowed (bfloat16). The float16
path rounds no operand: 0.75 u.
"""

import pytest
import torch

from nvsubquadratic_b200.decay_attention import decay_attention, decay_attention_step
from oracle.decay_attention import decay_attention as oracle_forward
from oracle.decay_attention import decay_attention_grads
from tests.conftest import rel_l2

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 128 * 2.0 ** -24, BF16: 1.5 * 2.0 ** -8, F16: 0.75 * 2.0 ** -11}


def _decays(H, kind):
    if kind == "spread":  # memories of 4 .. 4096 tokens
        return torch.log1p(-(2.0 ** -torch.linspace(2.0, 12.0, H, dtype=torch.float64))).float()
    if kind == "none":  # a = 1
        return torch.zeros(H)
    if kind == "strong":  # nothing is left after a few tokens; the last head forgets at once
        g = -torch.linspace(0.5, 40.0, H)
        g[-1] = float("-inf")
        return g
    raise ValueError(kind)


def _inputs(B, L, H, Hk, Dk, Dv, dtype, seed=0, decay="spread"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, v = r(B, L, H, Dk).to(dtype), r(B, L, Hk, Dk).to(dtype), r(B, L, Hk, Dv).to(dtype)
    return q, k, v, _decays(H, decay), r(B, H, Dk, Dv), r(B, L, H, Dv).to(dtype), r(B, H, Dk, Dv)


# ---------------------------------------------------------------- CPU


def test_oracle_gradients_are_differences():
    """Central differences of the float64 recurrence along random directions (it is linear in q, in k, in v and in the
    state, so those are exact up to rounding; log_decay: error O(eps^2))."""
    torch.manual_seed(0)
    q, k, v, g, s0, do, ds = _inputs(2, 9, 4, 2, 3, 5, F32)
    lengths = torch.tensor([9, 4], dtype=torch.int32)

    def loss(q, k, v, g, s0):
        o, s = oracle_forward(q, k, v, g, initial_state=s0, lengths=lengths)
        return ((o * do.double()).sum() + (s * ds.double()).sum()).item()

    args = [t.double() for t in (q, k, v, g, s0)]
    grads = decay_attention_grads(*args[:4], do, ds, initial_state=s0, lengths=lengths)
    eps = 1e-5
    for i in range(5):
        d = torch.randn_like(args[i])
        up, down = [list(args), list(args)]
        up[i], down[i] = args[i] + eps * d, args[i] - eps * d
        slope = (loss(*up) - loss(*down)) / (2 * eps)
        assert slope == pytest.approx((grads[i] * d).sum().item(), rel=1e-6, abs=1e-7), i


def test_refusals():
    q, k, v, g, s0, _, _ = _inputs(2, 5, 4, 2, 8, 6, F32)
    with pytest.raises(RuntimeError, match="CUDA"):
        decay_attention(q, k, v, g)
    with pytest.raises(AssertionError, match=r"\[B, L, heads, D\]"):
        decay_attention(q[0], k, v, g)
    with pytest.raises(AssertionError, match="must divide"):
        decay_attention(q[:, :, :3], k, v, g[:3])
    with pytest.raises(AssertionError, match="same heads"):
        decay_attention(q, k, v[:, :, :1], g)
    with pytest.raises(AssertionError, match="agree"):
        decay_attention(q[..., :7], k, v, g)
    with pytest.raises(AssertionError, match="agree"):
        decay_attention(q[:, :4], k, v, g)
    with pytest.raises(AssertionError, match="log_decay"):
        decay_attention(q, k, v, g[:3])
    with pytest.raises(AssertionError, match="share a dtype"):
        decay_attention(q.half(), k, v, g)
    with pytest.raises(NotImplementedError, match="float64"):
        decay_attention(q.double(), k.double(), v.double(), g)
    with pytest.raises(AssertionError, match="initial_state must be"):
        decay_attention(q, k, v, g, initial_state=s0[:1])
    with pytest.raises(AssertionError, match="float32"):
        decay_attention(q, k, v, g, initial_state=s0.half())
    with pytest.raises(AssertionError, match="lengths must be int32"):
        decay_attention(q, k, v, g, lengths=torch.tensor([1, 2]))
    with pytest.raises(AssertionError, match=r"lengths must be \[2\]"):
        decay_attention(q, k, v, g, lengths=torch.tensor([1], dtype=torch.int32))
    tok = (q[:, 0], k[:, 0], v[:, 0], g)
    with pytest.raises(AssertionError, match=r"\[B, heads, D\]"):
        decay_attention_step(q, k, v, g, s0)
    with pytest.raises(AssertionError, match="as many states"):
        decay_attention_step(*tok, s0[:1])
    with pytest.raises(AssertionError, match="contiguous"):
        decay_attention_step(*tok, s0.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(AssertionError, match="slots must be int32"):
        decay_attention_step(*tok, s0, slots=torch.tensor([0, 1]))
    with pytest.raises(NotImplementedError, match="no gradient"):
        decay_attention_step(q[:, 0].requires_grad_(), *tok[1:], s0)
    with pytest.raises(RuntimeError, match="CUDA"):
        decay_attention_step(q[:, 0].detach(), *tok[1:], s0)


def test_library_refuses_what_it_does_not_cover():
    import ctypes

    from nvsubquadratic_b200 import _lib

    def sizes(**kw):
        d = _lib.DecayDesc()
        for n, x in dict(dict(batch=1, heads=4, kv_heads=2, dk=64, dv=64, dtype=1, length=100, scale=1.0), **kw).items():
            setattr(d, n, x)
        f, b = ctypes.c_size_t(), ctypes.c_size_t()
        return _lib.load().hyfft_decay_workspace_size(ctypes.byref(d), ctypes.byref(f), ctypes.byref(b))

    assert sizes() == _lib.HYFFT_OK and sizes(length=0) == _lib.HYFFT_OK
    for bad in (dict(batch=0), dict(length=-1), dict(heads=0), dict(kv_heads=3), dict(dk=0), dict(dtype=3)):
        assert sizes(**bad) == _lib.HYFFT_ERR_INVALID, bad
    for bad in (dict(dk=257), dict(dv=300), dict(length=1 << 31)):
        assert sizes(**bad) == _lib.HYFFT_ERR_UNSUPPORTED, bad


# ---------------------------------------------------------------- GPU

# B, L, H, Hk, Dk, Dv
SHAPES = [
    (2, 1, 2, 2, 64, 64),
    (1, 31, 3, 1, 16, 16),
    (2, 33, 2, 2, 40, 72),
    (1, 127, 4, 2, 64, 64),
    (2, 129, 2, 1, 128, 128),
    (1, 300, 2, 2, 64, 128),
    (1, 300, 2, 2, 128, 64),
    (1, 77, 2, 1, 130, 7),
    (1, 70, 1, 1, 256, 200),
    (3, 65, 2, 2, 1, 1),
    (1, 1037, 2, 2, 48, 48),
]


def _run(q, k, v, g, s0, do, ds, lengths=None, learn=True):
    dev = [t.cuda().requires_grad_() for t in (q, k, v, g, s0)]
    dev[3].requires_grad_(learn)
    lengths = lengths.cuda() if lengths is not None else None
    o, s = decay_attention(*dev[:4], initial_state=dev[4], lengths=lengths, return_state=True)
    want = [t for t in dev if t.requires_grad]
    grads = list(torch.autograd.grad([o, s], want, [do.cuda(), ds.cuda()]))
    if not learn:
        grads.insert(3, None)
    return o, s, grads


def _compare(args, got, lengths=None, dtype=F32):
    q, k, v, g, s0, do, ds = args
    o, s, grads = got
    ro, rs = oracle_forward(q, k, v, g, initial_state=s0, lengths=lengths)
    ref = decay_attention_grads(q, k, v, g, do, ds, initial_state=s0, lengths=lengths)
    errs = {"o": rel_l2(ro, o)}
    for name, r, x in zip(("dq", "dk", "dv"), ref, grads):
        assert x.dtype == dtype
        errs[name] = rel_l2(r, x)
    assert o.dtype == dtype
    bad = {n: e for n, e in errs.items() if not e <= TOL[dtype]}
    # states and the decay's gradient are float32 whatever the inputs' type
    for name, r, x in (("state", rs, s), ("dlog_decay", ref[3], grads[3]), ("dstate", ref[4], grads[4])):
        if x is not None:
            assert x.dtype == F32
            e = rel_l2(r, x)
            if not e <= TOL[F32]:
                bad[name] = e
    assert not bad, bad


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype):
    args = _inputs(*shape, dtype)
    _compare(args, _run(*args), dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("decay", ["none", "strong"])
@pytest.mark.parametrize("shape", [(2, 150, 4, 2, 64, 64), (1, 700, 3, 3, 24, 40), (1, 260, 2, 2, 128, 128)], ids=str)
def test_decays_at_the_ends(shape, decay, dtype):
    args = _inputs(*shape, dtype, decay=decay)
    _compare(args, _run(*args), dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5, 260, 2, 1, 64, 64), (5, 1500, 2, 2, 64, 64), (5, 200, 2, 2, 128, 96)], ids=str)
def test_lengths_and_poisoned_padding(shape, dtype):
    """Lengths of none, one, ragged and all; NaN and infinities past them reach nothing, and nothing is left there."""
    args = list(_inputs(*shape, dtype))
    B, L = shape[:2]
    lengths = torch.tensor([L, 0, 1, L // 2 + 3, L - 1], dtype=torch.int32)
    past = (torch.arange(L)[None, :] >= lengths[:, None])
    poisoned = list(args)
    for i, bad in ((0, float("nan")), (1, float("inf")), (2, float("nan")), (5, float("-inf"))):
        t = args[i].clone()
        t[past] = bad
        poisoned[i] = t
    got = _run(*poisoned, lengths=lengths)
    _compare(args, got, lengths=lengths, dtype=dtype)
    for t in (got[0], *got[2][:3]):
        assert (t.cpu()[past] == 0).all()
    assert torch.equal(got[1][1].cpu(), args[4][1])  # no token: the state as it was
    assert torch.equal(got[2][4][1].cpu(), args[6][1])  # and its gradient


@gpu
def test_lengths_outside_the_sequence_are_clamped():
    args = _inputs(2, 40, 2, 2, 64, 64, F32)
    a = _run(*args, lengths=torch.tensor([-3, 1000], dtype=torch.int32))
    b = _run(*args, lengths=torch.tensor([0, 40], dtype=torch.int32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_strided_views_and_odd_alignment(D, dtype):
    """q, k, v as views of one projection, transposed heads, and rows that start off any 16-byte boundary."""
    B, L, H = 2, 150, 3
    args = _inputs(B, L, H, H, D, D, dtype)
    q, k, v, g, s0, do, ds = args
    want_o, want_s = oracle_forward(q, k, v, g, initial_state=s0)
    packed = torch.cat([t.flatten(2) for t in (q, k, v)], -1).cuda()
    views = [packed[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3)]
    heads = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        odd.append(flat[1:].view(t.shape).copy_(t))
    apart = [torch.stack((t, t), -1).flatten(-2).cuda()[..., ::2] for t in (q, k, v)]  # feature stride 2
    for form in (views, heads, odd, apart):
        o, s = decay_attention(*form, g.cuda(), initial_state=s0.cuda(), return_state=True)
        assert rel_l2(want_o, o) <= TOL[dtype] and rel_l2(want_s, s) <= TOL[F32]
    leaf = packed.clone().requires_grad_()
    q3 = [leaf[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3)]
    o = decay_attention(*q3, g.cuda())
    strided = torch.stack((do, do), 1).cuda()[:, 0]  # an upstream gradient with gaps between its batches
    (grad,) = torch.autograd.grad(o, [leaf], strided)
    ref = decay_attention_grads(q, k, v, g, do)
    assert rel_l2(torch.cat([t.flatten(2) for t in ref[:3]], -1), grad) <= TOL[dtype]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_empty_extents(dtype):
    q, k, v, g, s0, do, ds = (t.cuda() for t in _inputs(2, 0, 2, 2, 64, 64, dtype))
    s0.requires_grad_()
    o, s = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(s, s0)
    (ds0,) = torch.autograd.grad(s, [s0], ds)
    assert torch.equal(ds0, ds)
    o, s = decay_attention(q[:0], k[:0], v[:0], g, return_state=True)
    assert o.shape == (0, 0, 2, 64) and s.shape == (0, 2, 64, 64)
    assert decay_attention_step(q.new_empty(0, 2, 64), k.new_empty(0, 2, 64), v.new_empty(0, 2, 64), g,
                                s0.detach()).shape == (0, 2, 64)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_long_axis_and_split_sequences(D, dtype):
    """One row of 20000 tokens (many segments), and the same in two calls joined by the state."""
    L, cut = 20000, 7777
    q, k, v, g, s0, do, ds = _inputs(1, L, 2, 2, D, D, dtype)
    o, s = decay_attention(*(t.cuda() for t in (q, k, v, g)), return_state=True)
    ro, rs = oracle_forward(q, k, v, g)
    assert rel_l2(ro, o) <= TOL[dtype] and rel_l2(rs, s) <= TOL[F32]
    o1, s1 = decay_attention(*(t[:, :cut].cuda() for t in (q, k, v)), g.cuda(), return_state=True)
    o2, s2 = decay_attention(*(t[:, cut:].cuda() for t in (q, k, v)), g.cuda(), initial_state=s1, return_state=True)
    assert rel_l2(ro, torch.cat((o1, o2), 1)) <= TOL[dtype] and rel_l2(rs, s2) <= TOL[F32]


@gpu
def test_float32_gradients_are_differences():
    """Slopes of the kernel's own forward: it is linear in q, in k, in v and in the state, so a central difference with
    eps = 1 has no truncation error, only the forward's rounding (7.6e-6 of the loss's largest size on either side)."""
    args = _inputs(2, 200, 4, 2, 64, 48, F32)
    _, _, grads = _run(*args)
    base = [t.cuda() for t in args[:5]]
    do, ds = args[5].cuda().double(), args[6].cuda().double()
    for i in (0, 1, 2, 4):
        d = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        ends = []
        for sign in (1, -1):
            a = list(base)
            a[i] = a[i] + sign * d
            o, s = decay_attention(*a[:4], initial_state=a[4], return_state=True)
            ends.append((o.double() * do).sum() + (s.double() * ds).sum())
            size = o.double().norm() * do.norm() + s.double().norm() * ds.norm()
        slope = (ends[0] - ends[1]) / 2
        want = (grads[i].double() * d.double()).sum()
        assert abs(slope - want) <= 2 * TOL[F32] * size, (i, slope, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_same_bits_every_time(dtype):
    args = _inputs(2, 900, 4, 2, 64, 64, dtype)
    a, b = _run(*args), _run(*args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@gpu
def test_only_the_gradients_asked_for():
    q, k, v, g, s0, do, ds = (t.cuda() for t in _inputs(1, 100, 2, 1, 64, 64, BF16))
    full = _run(*(t.cpu() for t in (q, k, v, g, s0, do, ds)))[2]
    for i, t in enumerate((q, k, v, g, s0)):
        t.requires_grad_()
        o, s = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
        (grad,) = torch.autograd.grad([o, s], [t], [do, ds])
        assert torch.equal(grad, full[i])
        t.requires_grad_(False)
    s0.requires_grad_()  # the state alone
    _, s = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    (grad,) = torch.autograd.grad([s], [s0], [ds])
    assert rel_l2(ds.double() * torch.exp(100 * g.double())[None, :, None, None], grad) <= TOL[F32]


@gpu
def test_on_a_side_stream():
    args = _inputs(2, 500, 4, 4, 64, 64, BF16)
    want = _run(*args)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = _run(*args)
    st.synchronize()
    assert torch.equal(want[0], got[0]) and all(torch.equal(x, y) for x, y in zip(want[2], got[2]))


@gpu
def test_float16_states_beyond_its_range():
    """A state that grows past 65504 inside: the outputs fit float16 and are right."""
    L = 1000
    k = torch.full((1, L, 1, 64), 16.0, dtype=F16)
    v = torch.full((1, L, 1, 64), 16.0, dtype=F16)
    q = torch.full((1, L, 1, 64), 2.0 ** -12, dtype=F16)
    g = torch.zeros(1)
    o = decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), scale=1.0)
    assert rel_l2(oracle_forward(q, k, v, g, scale=1.0)[0], o) <= TOL[F16]


# B, H, Hk, Dk, Dv, pool
STEPS = [(1, 1, 1, 1, 1, 1), (1, 12, 12, 64, 64, 1), (5, 6, 2, 64, 64, 9), (3, 2, 2, 40, 72, 3), (2, 2, 1, 130, 7, 4),
         (40, 16, 16, 128, 128, 41), (2, 1, 1, 256, 256, 2), (3, 3, 3, 33, 31, 5)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", STEPS, ids=str)
def test_step(shape, dtype):
    B, H, Hk, Dk, Dv, N = shape
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    q, k, v, state = r(B, H, Dk).to(dtype), r(B, Hk, Dk).to(dtype), r(B, Hk, Dv).to(dtype), r(N, H, Dk, Dv)
    g = _decays(H, "spread")
    slots = torch.randperm(N, generator=gen)[:B].to(torch.int32)
    if B > 2:
        slots[1], slots[2] = -1, N  # idle requests
    live = (slots >= 0) & (slots < N)
    at = slots[live].long()
    ro, rs = oracle_forward(q[live, None], k[live, None], v[live, None], g, initial_state=state[at])
    want_o, want_s = torch.zeros(B, H, Dv, dtype=torch.float64), state.double()
    want_o[live], want_s[at] = ro[:, 0], rs
    dev = [t.cuda() for t in (q, k, v, g, state)]
    o = decay_attention_step(*dev, slots=slots.cuda())
    assert o.dtype == dtype and rel_l2(want_o, o) <= TOL[dtype]
    assert rel_l2(want_s, dev[4]) <= TOL[F32]
    idle = torch.ones(N, dtype=torch.bool)
    idle[at] = False
    assert torch.equal(dev[4].cpu()[idle], state[idle])  # rows that nobody owns
    assert (o.cpu()[~live] == 0).all()
    # into another buffer: the old states stay
    dev[4] = state.cuda()
    out = torch.full_like(dev[4], 7.0)
    o2 = decay_attention_step(*dev, slots=slots.cuda(), out_state=out)
    assert torch.equal(o, o2) and torch.equal(dev[4].cpu(), state)
    assert rel_l2(want_s[at], out.cpu()[at]) <= TOL[F32] and (out.cpu()[idle] == 7.0).all()


@gpu
def test_step_strided_inputs_and_unaligned_states():
    B, H, D = 3, 2, 64
    gen = torch.Generator().manual_seed(2)
    packed = torch.randn(B, 3 * H * D, generator=gen).to(BF16)
    q, k, v = (packed[:, i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    state = torch.randn(B, H, D, D, generator=gen)
    g = _decays(H, "spread")
    ro, rs = oracle_forward(q[:, None], k[:, None], v[:, None], g, initial_state=state)
    p = packed.cuda()
    q, k, v = (p[:, i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    flat = torch.empty(state.numel() + 1, device="cuda")
    s = flat[1:].view(state.shape).copy_(state)  # 4 bytes off a 16-byte boundary
    o = decay_attention_step(q, k, v, g.cuda(), s)
    assert rel_l2(ro[:, 0], o) <= TOL[BF16] and rel_l2(rs, s) <= TOL[F32]


@gpu
def test_steps_follow_the_sequence():
    """Token by token from a prompt's state gives what the sequence form gives."""
    B, L, H, D = 2, 90, 3, 64
    q, k, v, g, s0, _, _ = (t.cuda() for t in _inputs(B, L, H, H, D, D, F32))
    want, ws = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    o, s = decay_attention(q[:, :60], k[:, :60], v[:, :60], g, initial_state=s0, return_state=True)
    got = [o]
    for t in range(60, L):
        got.append(decay_attention_step(q[:, t], k[:, t], v[:, t], g, s).unsqueeze(1))
    assert rel_l2(want, torch.cat(got, 1)) <= 2 * TOL[F32] and rel_l2(ws, s) <= 2 * TOL[F32]


# ---------------------------------------------------------------- one rounding

# A bfloat16 value m 2^e, 1 <= m < 2, is off by a uniform error of spacing 2^(e-7): rms 2^(e-7) / sqrt(12), so a tensor that is
# rounded to nearest once is off by at most 2^-7 / sqrt(12) of its norm. What the scan itself rounds, it keeps in 16 bits
# (2^-17 of an operand); four times that is allowed beside.
ONE_ROUNDING = 2.0 ** -7 / 12 ** 0.5 + 2.0 ** -15

# uncut rows, cut ones, head sizes of both widths, shared heads
ROUNDED = [(40, 200, 4, 4, 64, 64), (40, 200, 4, 2, 128, 128), (2, 1500, 2, 1, 64, 64), (1, 1500, 2, 2, 128, 128),
           (1, 700, 2, 2, 96, 40)]


@gpu
@pytest.mark.parametrize("shape", ROUNDED, ids=str)
def test_bfloat16_results_are_rounded_once(shape):
    args = _inputs(*shape, BF16)
    o, _, grads = _run(*args, learn=False)
    q, k, v, g, s0, do, ds = args
    errs = {"o": rel_l2(oracle_forward(q, k, v, g, initial_state=s0)[0], o)}
    ref = decay_attention_grads(q, k, v, g, do, ds, initial_state=s0)
    errs.update({n: rel_l2(r, x) for n, r, x in zip(("dq", "dk", "dv"), ref, grads)})
    assert all(e <= ONE_ROUNDING for e in errs.values()), errs


# ---------------------------------------------------------------- waits that run out


def test_wait_limit_is_kept():
    from nvsubquadratic_b200 import _lib

    lib = _lib.load()
    before = lib.hyfft_set_wait_clocks(1000)
    assert lib.hyfft_set_wait_clocks(-1) == 1000 and lib.hyfft_set_wait_clocks(before) == 1000
    assert lib.hyfft_set_wait_clocks(-1) == before == 1 << 31


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(2, 700, 4, 2, 64, 64), (2, 700, 2, 2, 128, 128), (40, 300, 4, 4, 64, 64), (1, 300, 2, 2, 65, 33)],
                         ids=str)
def test_waits_that_run_out_leave_nan_and_a_status(shape, dtype):
    """With no patience at all some wait inside the tensor-core scan runs out: every value is the right one or NaN, the host
    can tell, and the next call is as ever."""
    from nvsubquadratic_b200 import _lib

    args = _inputs(*shape, dtype)
    want = _run(*args)
    _lib.check_waits(0)
    lib = _lib.load()
    before = lib.hyfft_set_wait_clocks(0)
    try:
        got = _run(*args)
        torch.cuda.synchronize()
    finally:
        lib.hyfft_set_wait_clocks(before)
    with pytest.raises(_lib.HyfftError, match="ran out"):
        _lib.check_waits(0)
    _lib.check_waits(0)  # it was cleared
    for a, b in zip((want[0], want[1], *want[2]), (got[0], got[1], *got[2])):
        assert ((a == b) | b.isnan()).all()
    assert got[0].isnan().any()
    again = _run(*args)
    for a, b in zip((want[0], want[1], *want[2]), (again[0], again[1], *again[2])):
        assert torch.equal(a, b)
    _lib.check_waits(0)


# ---------------------------------------------------------------- infinities and NaN in live tokens


def _same_kinds(name, want, got, tol):
    """NaN and infinities where float64 has them, and the rest right."""
    want, got = want.detach().double().cpu(), got.detach().double().cpu()
    assert torch.equal(want.isnan(), got.isnan()), name
    odd = want.isinf()
    assert torch.equal(odd, got.isinf()) and torch.equal(want[odd], got[odd]), name
    ok = want.isfinite()
    assert rel_l2(want[ok], got[ok]) <= tol, (name, rel_l2(want[ok], got[ok]))


@gpu
@pytest.mark.parametrize("where", ["q", "k", "v", "do", "state", "dstate"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")], ids=["inf", "nan"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(40, 150, 4, 2, 64, 64), (2, 600, 2, 2, 64, 72), (1, 530, 2, 1, 128, 128), (2, 30, 2, 2, 64, 64),
                                   (1, 90, 2, 2, 136, 20)], ids=str)
def test_bad_values_reach_what_the_recurrence_lets_them_reach(shape, dtype, bad, where):
    """One infinity or NaN in one live token: earlier tokens, other heads and other sequences are as if it were not there, and an
    infinity comes out as one. On either path, with the axis cut or not."""
    B, L, H, Hk, Dk, Dv = shape
    args = list(_inputs(*shape, dtype))
    i = ("q", "k", "v", None, "state", "do", "dstate").index(where)
    t = args[i].clone()
    if where in ("state", "dstate"):
        t[B - 1, 1, 3, 5] = bad
    else:
        t[B - 1, L * 2 // 3, -1, 5] = bad
    args[i] = t
    o, s, grads = _run(*args, learn=False)
    q, k, v, g, s0, do, ds = args
    ro, rs = oracle_forward(q, k, v, g, initial_state=s0)
    ref = decay_attention_grads(q, k, v, g, do, ds, initial_state=s0)
    _same_kinds("o", ro, o, TOL[dtype])
    _same_kinds("state", rs, s, TOL[F32])
    for n, r, x in zip(("dq", "dk", "dv"), ref, grads):
        _same_kinds(n, r, x, TOL[dtype])
    _same_kinds("dstate", ref[4], grads[4], TOL[F32])


@gpu
@pytest.mark.parametrize("shape", [(2, 100, 2, 2, 64, 64), (2, 20, 2, 2, 64, 64), (1, 600, 2, 1, 96, 40)], ids=str)
def test_float32_values_beyond_bfloat16(shape):
    """The largest float32 is finite, though it rounds to an infinity in 8 bits."""
    q, k, v, g, _, _, _ = _inputs(*shape, F32)
    q, k = q * 2.0 ** -40, k * 2.0 ** -4
    v[0, 30 if shape[1] > 30 else 5, 0, 5] = torch.finfo(F32).max
    v[0, 10, -1, 7] = -torch.finfo(F32).max
    o, s = decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), return_state=True)
    ro, rs = oracle_forward(q, k, v, g)
    for col in (5, 7, 9):  # the columns' sizes differ by 2^128
        assert rel_l2(ro[..., col], o[..., col]) <= TOL[F32] and rel_l2(rs[..., col], s[..., col]) <= TOL[F32]


@gpu
def test_second_and_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    q, k, v, g, s0, do, ds = (t.cuda() for t in _inputs(1, 40, 2, 1, 64, 64, F32))
    leaf = q.clone().requires_grad_()
    (dq,) = torch.autograd.grad(decay_attention(leaf, k, v, g).square().sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (leaf.sum() + dq.sum()).backward()
    args = [q, k, v, g]
    with forward_ad.dual_level():
        for i in range(5):
            a = list(args) + [s0]
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises((RuntimeError, NotImplementedError), match="forward mode AD"):
                decay_attention(*a[:4], initial_state=a[4])
        dual = forward_ad.make_dual(q[:, 0].contiguous(), torch.ones_like(q[:, 0]))
        with pytest.raises(NotImplementedError, match="no gradient"):
            decay_attention_step(dual, k[:, 0], v[:, 0], g, s0)
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0)


@gpu
def test_step_without_states():
    """A pool of no states: every request is idle."""
    q, k, v = (torch.randn(2, 3, 16, device="cuda") for _ in range(3))
    state = torch.empty(0, 3, 16, 16, device="cuda")
    o = decay_attention_step(q, k, v, torch.zeros(3, device="cuda"), state, slots=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert o.shape == (2, 3, 16) and (o == 0).all()


# ---------------------------------------------------------------- buffers that are used many times over

# Rows that fill the machine and are walked whole (16 chunks and more of 64 tokens), few of them in segments of two dozen chunks,
# and head sizes of two column slices whose axis is cut. Checked on some of the batch, which the float64 recurrence can afford.
LONG = [
    (16, 1023, 12, 4, 64, 64),
    (38, 700, 4, 4, 128, 96),
    (40, 650, 4, 2, 72, 64),
    (25, 3000, 4, 4, 64, 64),
    (25, 3000, 2, 2, 128, 128),
    (10, 2600, 4, 2, 96, 128),
    (1, 1500, 2, 2, 128, 128),
    (2, 900, 2, 1, 96, 72),
    (1, 1100, 3, 3, 80, 128),
    (1, 1037, 4, 2, 100, 100),
]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_many_chunks(shape, dtype):
    B, L = shape[:2]
    args = _inputs(*shape, dtype)
    lengths = None
    if B > 1:
        lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(5), dtype=torch.int32)
        lengths[0], lengths[-1] = L, L - 1
    o, s, grads = _run(*args, lengths=lengths, learn=False)
    some = torch.tensor([0, B - 1] if L > 2000 else sorted({0, B // 2, B - 1}))
    q, k, v, g, s0, do, ds = args
    part = [t[some] for t in (q, k, v)] + [g] + [t[some] for t in (s0, do, ds)]
    got = (o.cpu()[some], s.cpu()[some], [t.cpu()[some] if t is not None else None for t in grads])
    _compare(part, got, lengths=lengths[some] if lengths is not None else None, dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(2, 20, 2, 2, 3, 5), (2, 100, 2, 1, 5, 3), (1, 40, 1, 1, 129, 2), (1, 40, 1, 1, 2, 131)], ids=str)
def test_infinities_of_heads_smaller_than_their_tiles(shape, dtype):
    """All else positive, so that the recurrence keeps the sign of an infinity in v or do: the places that pad a head count for nothing."""
    args = [t.abs() if t.ndim > 1 else t for t in _inputs(*shape, dtype)]
    for i in (2, 5):
        bad = list(args)
        bad[i] = args[i].clone()
        bad[i][0, 7, 0, 1] = float("-inf")
        q, k, v, g, s0, do, ds = bad
        o, s, grads = _run(*bad, learn=False)
        ro, rs = oracle_forward(q, k, v, g, initial_state=s0)
        ref = decay_attention_grads(q, k, v, g, do, ds, initial_state=s0)
        assert (ro.isinf() if i == 2 else ref[0].isinf()).any()
        _same_kinds("o", ro, o, TOL[dtype])
        _same_kinds("state", rs, s, TOL[F32])
        for n, r, x in zip(("dq", "dk", "dv"), ref, grads):
            _same_kinds(n, r, x, TOL[dtype])
        _same_kinds("dstate", ref[4], grads[4], TOL[F32])
