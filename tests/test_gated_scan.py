"""Gated linear recurrence: the oracle and refusals (CPU); sequences, their gradients and single tokens against the float64
oracle (GPU).

Tolerances (relative L2). In float32 a decay's complement is off by 16 * 2^-24 of itself at most (|gate| <= 8 here: the exponential 2 +
1.2 |gate| units, a division 2, a product 1), and a state or a gradient of the state, whose weights are products of decays that
forget as much as they have gathered, by three times that; with the roundings of its sums 64 * 2^-24. A gradient of a gate multiplies a
state with a gradient: 128 * 2^-24 for all. 16-bit outputs are rounded once more, by at most 2^-8 of an element in bfloat16 and 2^-11 in
float16, where an element below 2^-14 is off by 2^-25 instead.
"""

import pytest
import torch

from nvsubquadratic_b200.gated_scan import gated_scan, gated_scan_step
from oracle.gated_scan import gated_scan as oracle

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 128 * 2.0 ** -24, BF16: 2.0 ** -8 + 128 * 2.0 ** -24, F16: 2.0 ** -11 + 128 * 2.0 ** -24}
DTYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
FORMS = pytest.mark.parametrize("form", ["logit", "log"])


def close(want, got, dtype, times=1.0):
    want, got = want.detach().double().cpu(), got.detach().double().cpu()
    assert want.shape == got.shape
    floor = 2.0 ** -25 * want.numel() ** 0.5 if dtype is F16 else 0.0
    err = torch.linalg.norm(want - got).item()
    assert err <= times * TOL[dtype] * torch.linalg.norm(want).item() + floor, err / max(want.norm().item(), 1e-30)


def _gate(g, shape, form, dtype, most=8.0):
    if form == "logit":
        return (2 + 2 * torch.randn(shape, generator=g)).clamp(-most, most).to(dtype)
    return (-torch.exp(1.5 * torch.randn(shape, generator=g) - 3)).clamp(min=-most).to(dtype)


def _case(B, L, C, dtype, form="logit", out_gate=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(x=r(B, L, C).to(dtype), gate=_gate(g, (B, L, C), form, dtype), out_gate=r(B, L, C).to(dtype) if out_gate else None,
                initial_state=r(B, C), dy=r(B, L, C).to(dtype), dstate=r(B, C))


# ---------------------------------------------------------------- CPU


@pytest.mark.parametrize("complement", [True, False])
@FORMS
@pytest.mark.parametrize("with_gate", [True, False])
def test_oracle_gradients_are_autograds(form, complement, with_gate):
    c = _case(2, 9, 3, torch.float64, form, with_gate)
    lengths = [9, 5]
    leaves = {k: c[k].double().requires_grad_() for k in ("x", "gate", "out_gate", "initial_state") if c[k] is not None}
    a = torch.sigmoid(leaves["gate"]) if form == "logit" else leaves["gate"].exp()
    h, ys, last = leaves["initial_state"], [], []
    for t in range(9):
        h = a[:, t] * h + ((1 - a[:, t]) if complement else 1) * leaves["x"][:, t]
        ys.append(h * torch.nn.functional.silu(leaves["out_gate"][:, t]) if with_gate else h)
        last.append(h)
    y, state = torch.stack(ys, 1), torch.stack([last[8][0], last[4][1]])
    y = torch.stack([y[0], torch.cat((y[1, :5], torch.zeros(4, 3, dtype=torch.float64)))])
    want = torch.autograd.grad([y, state], list(leaves.values()), [c["dy"], c["dstate"].double()])
    got = oracle(c["x"], c["gate"], c["out_gate"], form, complement, c["initial_state"], lengths, c["dy"], c["dstate"])
    assert torch.allclose(got[0], y) and torch.allclose(got[1], state)
    for w, o in zip(want, [got[2], got[3]] + ([got[4]] if with_gate else []) + [got[5]]):
        assert torch.allclose(w, o, atol=1e-12)


def test_refusals():
    x = torch.randn(2, 3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan(x, x)
    with pytest.raises(AssertionError, match="x must be"):
        gated_scan(x[0], x[0])
    with pytest.raises(AssertionError, match="gate must be"):
        gated_scan(x, x[:, :2])
    with pytest.raises(AssertionError, match="out_gate must be"):
        gated_scan(x, x, out_gate=x[..., :4])
    with pytest.raises(AssertionError, match="share a dtype"):
        gated_scan(x, x.half())
    with pytest.raises(ValueError, match="unknown form"):
        gated_scan(x, x, form="exp")
    with pytest.raises(NotImplementedError, match="float64"):
        gated_scan(x.double(), x.double())
    with pytest.raises(AssertionError, match="initial_state must be"):
        gated_scan(x, x, initial_state=torch.zeros(2, 7))
    with pytest.raises(AssertionError, match="initial_state must be float32"):
        gated_scan(x, x, initial_state=torch.zeros(2, 8).double())
    with pytest.raises(AssertionError, match="lengths must be"):
        gated_scan(x, x, lengths=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(AssertionError, match="int32"):
        gated_scan(x, x, lengths=torch.zeros(2, dtype=torch.int64))
    t, s = x[:, 0], torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan_step(t, t, s)
    with pytest.raises(AssertionError, match="need as many states"):
        gated_scan_step(t, t, s[:1])
    with pytest.raises(AssertionError, match="state must be"):
        gated_scan_step(t, t, s[0])
    with pytest.raises(AssertionError, match="out_state must be"):
        gated_scan_step(t, t, s, out_state=s[:2])
    with pytest.raises(AssertionError, match="contiguous"):
        gated_scan_step(t, t, torch.zeros(8, 4).t())
    with pytest.raises(AssertionError, match="slots must be int32"):
        gated_scan_step(t, t, s, slots=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(AssertionError, match=r"slots must be \[2\]"):
        gated_scan_step(t, t, s, slots=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(NotImplementedError, match="no gradient"):
        gated_scan_step(t.clone().requires_grad_(), t, s)


def test_library_refusals():
    """At the C entry, on the host, before anything is launched."""
    import ctypes

    from nvsubquadratic_b200 import _lib

    lib, p, size = _lib.load(), ctypes.c_void_p(16), ctypes.c_size_t()

    def desc(**kw):
        d = _lib.GatedDesc()
        d.batch, d.length, d.channels, d.dtype = 2, 20, 8, _lib.BF16
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    assert lib.hyfft_gated_saved_size(desc(), ctypes.byref(size)) == 0 and size.value == 4 * 2 * 3 * 8
    for bad in (dict(batch=0), dict(length=0), dict(channels=0), dict(dtype=3), dict(form=2)):
        assert lib.hyfft_gated_saved_size(desc(**bad), ctypes.byref(size)) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_gated_saved_size(desc(length=1 << 31), ctypes.byref(size)) == _lib.HYFFT_ERR_UNSUPPORTED
    assert lib.hyfft_gated_saved_size(None, ctypes.byref(size)) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_gated_forward(desc(), None, p, None, None, None, p, None, None, 0, None) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_gated_forward(desc(), p, p, None, None, None, p, None, p, 8, None) == _lib.HYFFT_ERR_WORKSPACE
    args = [p, p, None, None]
    assert lib.hyfft_gated_backward(desc(), *args, None, 0, p, None, p, p, None, None, None) == _lib.HYFFT_ERR_WORKSPACE
    args[2] = p  # an output gate without a place for its gradient
    assert lib.hyfft_gated_backward(desc(), *args, p, 1 << 20, p, None, p, p, None, None, None) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_gated_step(desc(), p, p, None, None, 1, p, p, p, None) == _lib.HYFFT_ERR_INVALID  # two requests, one state


# ---------------------------------------------------------------- GPU

# B, L, C: single tokens and channels, tiles and segments cut in every place, columns of 128 bytes cut, rows on and off 16 bytes
SHAPES = [(1, 1, 1), (2, 7, 3), (1, 8, 64), (3, 9, 65), (2, 63, 66), (1, 64, 72), (2, 65, 128), (2, 200, 40), (1, 515, 33),
          (4, 129, 130), (1, 1500, 24)]


def _run(c, form, complement, lengths=None, grads=True):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    leaves = {k: c[k].cuda().requires_grad_(grads) for k in ("x", "gate", "out_gate", "initial_state") if c[k] is not None}
    y, state = gated_scan(leaves["x"], leaves["gate"], out_gate=leaves.get("out_gate"), form=form, complement=complement,
                          initial_state=leaves.get("initial_state"), lengths=n, return_state=True)
    if not grads:
        return y, state
    return y, state, *torch.autograd.grad([y, state], list(leaves.values()), [c["dy"].cuda(), c["dstate"].cuda()])


def _want(c, form, complement, lengths=None):
    out = oracle(c["x"], c["gate"], c["out_gate"], form, complement, c["initial_state"], lengths, c["dy"], c["dstate"])
    out = [t for t in out if t is not None]
    return out if c["initial_state"] is not None else out[:-1]


@gpu
@pytest.mark.parametrize("complement,with_gate", [(True, True), (False, False), (True, False), (False, True)])
@FORMS
@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype, form, complement, with_gate):
    c = _case(*shape, dtype, form, with_gate)
    for i, (want, got) in enumerate(zip(_want(c, form, complement), _run(c, form, complement))):
        state = i == 1 or (i == 4 + with_gate)  # states and their gradients are float32
        assert got.dtype == (F32 if state else dtype)
        close(want, got, got.dtype)
    y, s = _run(c, form, complement, grads=False)
    full = _run(c, form, complement)
    assert torch.equal(y, full[0]) and torch.equal(s, full[1])  # with and without a gradient to come, bit for bit


@gpu
@DTYPES
@pytest.mark.parametrize("C", [64, 67])
def test_lengths(dtype, C):
    """Padding is neither read nor counted: it holds NaN here. Lengths outside 0 .. L are clamped."""
    B, L = 7, 150
    lengths = [150, 0, 1, 64, 65, 200, -3]
    c = _case(B, L, C, dtype)
    for k in ("x", "gate", "out_gate", "dy"):
        for b, n in enumerate(lengths):
            c[k][b, max(n, 0):] = float("nan")
    got = _run(c, "logit", True, lengths)
    clean = {k: torch.nan_to_num(v) for k, v in c.items()}
    for want, g in zip(_want(clean, "logit", True, lengths), got):
        close(want, g, g.dtype)
    for g in (got[0], *got[2:5]):
        for b, n in enumerate(lengths):
            assert (g[b, max(n, 0):] == 0).all()
    assert torch.equal(got[1][1].cpu(), c["initial_state"][1]) and torch.equal(got[5][1].cpu(), c["dstate"][1])


@gpu
def test_without_initial_state_and_partial_gradients():
    c = _case(2, 40, 10, F32)
    c["initial_state"] = None
    for want, got in zip(_want(c, "logit", True), _run(c, "logit", True)):
        close(want, got, F32)
    x, g = c["x"].cuda(), c["gate"].cuda().requires_grad_()
    y, state = gated_scan(x, g, return_state=True)
    want = oracle(c["x"], c["gate"], dy=c["dy"])
    (dg,) = torch.autograd.grad(y, [g], c["dy"].cuda(), retain_graph=True)
    close(want[3], dg, F32)
    want = oracle(c["x"], c["gate"], dy=torch.zeros_like(c["dy"]), dstate=c["dstate"])
    (dg,) = torch.autograd.grad(state, [g], c["dstate"].cuda())
    close(want[3], dg, F32)
    assert gated_scan(x, c["gate"].cuda()).dtype == F32  # no state asked for


@gpu
def test_gradients_are_the_slopes():
    """A gradient times a direction is the central difference of the float64 oracle along it (truncation 1e-6 of the third
    derivative, float32 gradients)."""
    c = _case(2, 90, 5, F32)
    got = _run(c, "logit", True)[2:]
    g = torch.Generator().manual_seed(1)
    for k, grad in zip(("x", "gate", "out_gate", "initial_state"), got):
        d, ends, eps = torch.randn(c[k].shape, generator=g).double(), [], 1e-4
        for sign in (1, -1):
            m = {n: t.double() for n, t in c.items()}
            m[k] = m[k] + sign * eps * d
            y, s = oracle(m["x"], m["gate"], m["out_gate"], initial_state=m["initial_state"])
            ends.append((y * m["dy"]).sum() + (s * m["dstate"]).sum())
        slope, have = ((ends[0] - ends[1]) / (2 * eps)).item(), (grad.double().cpu() * d).sum().item()
        assert abs(slope - have) <= 1e-5 * grad.double().norm().item() * d.norm().item()


@gpu
@DTYPES
def test_views_strides_and_alignment(dtype):
    B, L, C = 2, 70, 64
    c = _case(B, L, C, dtype)
    want = _want(c, "logit", True)
    names = ("x", "gate", "out_gate")
    packed = torch.cat([c[k] for k in names], -1).cuda()
    forms = [[packed[..., i * C:(i + 1) * C] for i in range(3)],                                     # one projection
             [c[k].transpose(0, 1).contiguous().cuda().transpose(0, 1) for k in names],               # tokens first
             [c[k].transpose(1, 2).contiguous().cuda().transpose(1, 2) for k in names],               # channels apart
             [torch.empty(B * L * C + 1, dtype=dtype, device="cuda")[1:].view(B, L, C).copy_(c[k]) for k in names],
             [torch.nn.functional.pad(c[k], (1, 2)).cuda()[..., 1:-2] for k in names]]                # odd rows
    for form in forms:
        leaves = [t.detach().requires_grad_() for t in form]
        y = gated_scan(leaves[0], leaves[1], out_gate=leaves[2], initial_state=c["initial_state"].cuda())
        dy = torch.nn.functional.pad(c["dy"], (3, 0)).cuda()[..., 3:]
        grads = torch.autograd.grad(y, leaves, dy)
        close(want[0], y, dtype)
        only = oracle(c["x"], c["gate"], c["out_gate"], initial_state=c["initial_state"], dy=c["dy"])
        for w, g in zip(only[2:5], grads):
            close(w, g, dtype)


@gpu
def test_broadcast_inputs_sum_their_gradients():
    """A gate shared by the batch and by all tokens: read in place, its gradient the sum of what it is spread over."""
    c = _case(3, 50, 16, F32, out_gate=False)
    gate = c["gate"][:1, :1].clone()
    leaf = gate.cuda().requires_grad_()
    x = c["x"].cuda().requires_grad_()
    y = gated_scan(x, leaf.expand(3, 50, 16))
    dx, dg = torch.autograd.grad(y, [x, leaf], c["dy"].cuda())
    want = oracle(c["x"], gate.expand(3, 50, 16), dy=c["dy"])
    close(want[0], y, F32)
    close(want[2], dx, F32)
    # 150 terms of either sign, each off by TOL of itself
    assert (want[3].sum((0, 1)) - dg[0, 0].double().cpu()).abs().max() <= TOL[F32] * want[3].abs().sum((0, 1)).max()


@gpu
@FORMS
@pytest.mark.parametrize("L", [4096, 20000])
def test_slow_decays_over_long_sequences(L, form):
    """One decay near 1 throughout, whose rounding would be raised to the power of the distance (4e-8 * 16384 for a memory of that
    many tokens). The exponential of a logit near -10 is off by 14 units."""
    c = _case(1, L, 8, F32, form, out_gate=False)
    memory = torch.tensor([30.0, 100, 400, 1000, 3000, 6000, 10000, 16384])
    c["gate"] = (torch.log(memory - 1) if form == "logit" else -1 / memory).expand(1, L, 8).contiguous()
    for want, got in zip(_want(c, form, True), _run(c, form, True)):
        for ch in range(8):
            close(want[..., ch], got[..., ch], F32)


@gpu
@FORMS
@pytest.mark.parametrize("L", [60, 300])
def test_infinities_and_nan_stay_where_the_recurrence_lets_them(L, form):
    c = _case(2, L, 8, F32, form)
    c["gate"][0, :, 0] = 8.0 if form == "logit" else -3e-4
    c["x"][0, L // 2, 0] = float("inf")
    c["x"][0, L // 2, 1] = float("nan")
    c["gate"][0, L // 3, 2] = float("nan")
    c["x"][1, L // 2, 3] = -float("inf")
    c["gate"][1, L // 2 + 1:, 3] = -8.0  # forgets so fast that its decays' product underflows; the infinity stays all the same
    c["gate"][1, 5:, 4] = -float("inf")  # a decay of zero: each token alone
    c["x"][1, 20, 5] = float("inf")
    c["gate"][1, 40, 5] = -float("inf")  # zero times infinity
    c["initial_state"][1, 6] = float("inf")
    want, got = _want(c, form, True), _run(c, form, True)
    for i in (0, 1):
        w, g = want[i], got[i].double().cpu()
        assert torch.equal(torch.isnan(w), torch.isnan(g))
        assert torch.equal(torch.isposinf(w), torch.isposinf(g)) and torch.equal(torch.isneginf(w), torch.isneginf(g))
        fine = torch.isfinite(w)
        close(w[fine], g[fine], F32)
    c["dy"][0, L // 2, 6] = float("inf")
    c["dy"][0, L // 2, 7] = float("nan")
    c["x"], c["gate"] = _case(2, L, 8, F32, form)["x"], _case(2, L, 8, F32, form)["gate"]
    c["initial_state"] = _case(2, L, 8, F32, form)["initial_state"]
    for w, g in zip(_want(c, form, True)[2:], _run(c, form, True)[2:]):
        g = g.double().cpu()
        assert torch.equal(torch.isnan(w), torch.isnan(g)) and torch.equal(torch.isinf(w), torch.isinf(g))
        fine = torch.isfinite(w)
        close(w[fine], g[fine], F32)


@gpu
def test_growing_log_decays():
    """Exponentials above 1 are taken as they are."""
    c = _case(1, 130, 4, F32, "log", out_gate=False)
    c["gate"] = (0.02 * torch.randn(1, 130, 4) + 0.01)
    for want, got in zip(_want(c, "log", False), _run(c, "log", False)):
        close(want, got, F32)


@gpu
def test_decays_above_one_whose_product_overflows():
    """exp(3) for each token: a state of zero stays zero however long, and what is put in grows as far as float32 goes."""
    L = 400
    x, g = torch.zeros(1, L, 8, device="cuda"), torch.full((1, L, 8), 3.0, device="cuda")
    y, s = gated_scan(x, g, form="log", complement=False, return_state=True)
    assert (y == 0).all() and (s == 0).all()
    x[0, 380, 1] = 1.0
    y, s = gated_scan(x, g, form="log", complement=False, return_state=True)
    want, end = oracle(x, g, form="log", complement=False)
    for ch in range(8):
        close(want[..., ch], y[..., ch], F32)
    close(end, s, F32)
    x[0, 100, 2] = 1.0
    y = gated_scan(x, g, form="log", complement=False)
    assert (y[0, :100, 2] == 0).all() and (y[0, 200:, 2] == float("inf")).all()
    assert (y[..., 3:] == 0).all() and torch.isfinite(y[..., :2]).all()


@gpu
def test_a_sequence_in_pieces_is_the_sequence():
    c = _case(2, 200, 48, F32)
    x, g, o = (c[k].cuda() for k in ("x", "gate", "out_gate"))
    want, end = gated_scan(x, g, out_gate=o, return_state=True)
    state, parts = None, []
    for a, b in ((0, 70), (70, 71), (71, 200)):
        y, state = gated_scan(x[:, a:b], g[:, a:b], out_gate=o[:, a:b], initial_state=state, return_state=True)
        parts.append(y)
    close(want, torch.cat(parts, 1), F32)
    close(end, state, F32)


@gpu
def test_empty_batches_and_sequences():
    x = torch.randn(0, 5, 8, device="cuda", requires_grad=True)
    y, s = gated_scan(x, x, return_state=True)
    assert y.shape == (0, 5, 8) and s.shape == (0, 8)
    torch.autograd.grad(y.sum(), [x])
    x, h = torch.randn(2, 0, 8, device="cuda"), torch.randn(2, 8, device="cuda", requires_grad=True)
    y, s = gated_scan(x, x, initial_state=h, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(s, h)
    (dh,) = torch.autograd.grad(s, [h], torch.ones_like(s))
    assert (dh == 1).all()
    assert (gated_scan(x, x, return_state=True)[1] == 0).all()


@gpu
def test_second_and_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    x = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(gated_scan(x, x).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    x = x.detach()
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward mode AD"):
            gated_scan(forward_ad.make_dual(x, torch.ones_like(x)), x)


@gpu
def test_streams_and_graphs():
    """Calls on a stream of their own, two at once, and a captured training step that is replayed with new inputs."""
    c = _case(3, 333, 96, BF16)
    args = [c[k].cuda() for k in ("x", "gate", "out_gate")]
    want = gated_scan(args[0], args[1], out_gate=args[2])
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(gated_scan(args[0], args[1], out_gate=args[2]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)

    leaves, dy = [a.clone().requires_grad_() for a in args], c["dy"].cuda()

    def step():
        return torch.autograd.grad(gated_scan(leaves[0], leaves[1], out_gate=leaves[2]), leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    other = _case(3, 333, 96, BF16, seed=1)
    with torch.no_grad():
        for leaf, k in zip(leaves, ("x", "gate", "out_gate")):
            leaf.copy_(other[k])
    graph.replay()
    torch.cuda.synchronize()
    kept = [g.clone() for g in got]
    for a, b in zip(kept, step()):
        assert torch.equal(a, b)


@gpu
@DTYPES
def test_more_rows_than_the_machine_runs_at_once(dtype):
    """Rows that one CTA each takes from end to end (few rows share theirs among several)."""
    B, L, C = 40, 150, 2048
    c = _case(B, L, C, dtype)
    some = torch.randint(0, C, (40,), generator=torch.Generator().manual_seed(2))
    few = {k: t[..., some] for k, t in c.items()}
    for want, got in zip(_want(few, "logit", True), _run(c, "logit", True)):
        close(want, got[..., some.cuda()], got.dtype)


@gpu
@pytest.mark.parametrize("C", [2048, 2101])
@DTYPES
def test_rows_that_clusters_share(dtype, C):
    """Rows enough to be 128 bytes wide and few enough for several CTAs each; ragged, on and off 16 bytes."""
    B, L, lengths = 3, 333, [333, 64, 200]
    if dtype is F32:
        C //= 2
    c = _case(B, L, C, dtype)
    some = torch.randint(0, C, (30,), generator=torch.Generator().manual_seed(2))
    some[:2] = torch.tensor([0, C - 1])
    few = {k: t[..., some] for k, t in c.items()}
    for want, got in zip(_want(few, "logit", True, lengths), _run(c, "logit", True, lengths)):
        close(want, got[..., some.cuda()], got.dtype)


@gpu
def test_waits_that_run_out():
    """A CTA that gives up on its neighbour's message leaves NaN from there on and a status for the host; the next call is sound."""
    from nvsubquadratic_b200 import _lib

    c = _case(2, 3000, 64, BF16)
    want = _run(c, "logit", True)
    _lib.check_waits(0)
    lib = _lib.load()
    before = lib.hyfft_set_wait_clocks(0)
    try:
        got = _run(c, "logit", True)
        torch.cuda.synchronize()
    finally:
        lib.hyfft_set_wait_clocks(before)
    if any(t.isnan().any() for t in got):
        with pytest.raises(_lib.HyfftError, match="gated scan"):
            _lib.check_waits(0)
    _lib.check_waits(0)
    for i in (0, 1):  # a message that came in time is the one that it is otherwise
        assert ((got[i] == want[i]) | got[i].isnan()).all()
    assert all(torch.equal(p, q) for p, q in zip(want, _run(c, "logit", True)))
    _lib.check_waits(0)


# ---------------------------------------------------------------- single tokens


@gpu
@pytest.mark.parametrize("with_gate", [True, False])
@FORMS
@DTYPES
@pytest.mark.parametrize("C", [1, 33, 64, 770])
def test_step(C, dtype, form, with_gate):
    B, N = 5, 9
    c = _case(B, 1, C, dtype, form, with_gate)
    x, g = c["x"][:, 0].cuda(), c["gate"][:, 0].cuda()
    o = c["out_gate"][:, 0].cuda() if with_gate else None
    pool = torch.randn(N, C, generator=torch.Generator().manual_seed(3))
    slots = [4, -1, 8, 0, 9]
    for complement in (True, False):
        want, state = oracle(c["x"], c["gate"], c["out_gate"], form, complement, pool[[4, 4, 8, 0, 0]])
        held, before = pool.cuda(), pool.cuda()
        x[1] = float("nan")  # idle: not read
        y = gated_scan_step(x, g, held, out_gate=o, form=form, complement=complement,
                            slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
        assert (y[[1, 4]] == 0).all()
        close(want[[0, 2, 3], 0], y[[0, 2, 3]], dtype)
        close(state[[0, 2, 3]], held[[4, 8, 0]], F32)
        rest = [1, 2, 3, 5, 6, 7]
        assert torch.equal(held[rest], before[rest])
        x[1] = c["x"][1, 0].cuda()
        new = torch.zeros_like(held)
        y = gated_scan_step(x, g, before, out_gate=o, form=form, complement=complement, out_state=new)
        want, state = oracle(c["x"], c["gate"], c["out_gate"], form, complement, pool[:B])
        close(want[:, 0], y, dtype)
        close(state, new[:B], F32)
        assert (new[B:] == 0).all() and torch.equal(before.cpu(), pool)


@gpu
def test_step_follows_the_sequence_and_reads_views():
    c = _case(4, 30, 64, F32)
    x, g, o = (c[k].cuda() for k in ("x", "gate", "out_gate"))
    want, end = gated_scan(x, g, out_gate=o, return_state=True)
    state = torch.zeros(4, 64, device="cuda")
    for t in range(30):
        close(want[:, t], gated_scan_step(x[:, t], g[:, t], state, out_gate=o[:, t]), F32)
    close(end, state, F32)
    empty = torch.zeros(0, 64, device="cuda")
    assert gated_scan_step(empty, empty, state).shape == (0, 64)
    idle = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    assert (gated_scan_step(x[:, 0], g[:, 0], empty, slots=idle) == 0).all()


@gpu
@pytest.mark.parametrize("B,L,C", [(2, 3000, 64), (3, 3000, 2048)], ids=["rows of 64 bytes", "rows of 128 bytes"])
def test_a_wait_that_runs_out_is_told(B, L, C):
    """With no patience at all some wait does run out: results and gradients are NaN from there on and what they are otherwise before,
    the status says so once, and the calls after it are sound."""
    from nvsubquadratic_b200 import _lib

    c = _case(B, L, C, BF16)
    want = _run(c, "logit", True)
    _lib.check_waits(0)
    lib, told = _lib.load(), 0
    before = lib.hyfft_set_wait_clocks(0)
    try:
        for _ in range(20):
            got = _run(c, "logit", True)
            torch.cuda.synchronize()
            for w, g in zip(want, got):
                assert ((g == w) | g.isnan()).all()
            if any(g.isnan().any() for g in got):
                with pytest.raises(_lib.HyfftError, match="gated scan"):
                    _lib.check_waits(0)
                told += 1
            _lib.check_waits(0)
    finally:
        lib.hyfft_set_wait_clocks(before)
    assert told > 0
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(want, _run(c, "logit", True)))
    _lib.check_waits(0)


@pytest.mark.parametrize("length", [0, -1, 1 << 40])
def test_the_length_of_a_steps_descriptor_is_not_used(length):
    """The C entry goes on to what it does look at: here two requests and one state, and no output."""
    import ctypes

    from nvsubquadratic_b200 import _lib

    lib, p, d = _lib.load(), ctypes.c_void_p(16), _lib.GatedDesc()
    d.batch, d.channels, d.dtype, d.length = 2, 8, _lib.F32, length
    assert lib.hyfft_gated_step(ctypes.byref(d), p, p, None, None, 1, p, p, p, None) == _lib.HYFFT_ERR_INVALID
    assert b"too few states" in lib.hyfft_last_error()
    assert lib.hyfft_gated_step(ctypes.byref(d), p, p, None, None, 2, p, p, None, None) == _lib.HYFFT_ERR_INVALID
    assert b"null tensor" in lib.hyfft_last_error()


@gpu
def test_a_step_through_the_c_entry_without_a_length():
    import ctypes

    from nvsubquadratic_b200 import _lib

    c = _case(3, 1, 8, F32)
    x, g, state, y = c["x"][:, 0].cuda(), c["gate"][:, 0].cuda(), c["initial_state"].cuda(), torch.empty(3, 8, device="cuda")
    d = _lib.GatedDesc()  # all zeros but what the step reads
    d.batch, d.channels, d.dtype, d.complement = 3, 8, _lib.F32, 1
    d.x_stride[0] = d.gate_stride[0] = 8
    rc = _lib.load().hyfft_gated_step(ctypes.byref(d), x.data_ptr(), g.data_ptr(), None, None, 3, state.data_ptr(), state.data_ptr(),
                                      y.data_ptr(), _lib.stream_ptr(x.device))
    _lib.check(rc, "hyfft_gated_step")
    want, end = oracle(c["x"], c["gate"], initial_state=c["initial_state"])
    close(want[:, 0], y, F32)
    close(end, state, F32)


@gpu
@FORMS
@DTYPES
@pytest.mark.parametrize("B,L,C,copies", [(1, 9003, 40, 1), (2, 3001, 40, 40)], ids=["rows of 64 bytes", "rows of 128 bytes"])
def test_long_rows_that_many_CTAs_take_in_turn(B, L, C, copies, dtype, form):
    """Tens of tiles for each CTA of a cluster, with output gates, states at both ends and every gradient; many rows are copies."""
    c = _case(B, L, C, dtype, form)
    lengths = [L, 2 * L // 3][:B]
    wide = {k: t.repeat(*[1] * (t.ndim - 1), copies) for k, t in c.items()}
    for want, got in zip(_want(c, form, True, lengths), _run(wide, form, True, lengths)):
        got = got.unflatten(-1, (copies, C))
        assert torch.equal(got, got[..., :1, :].expand_as(got))
        close(want, got[..., 0, :], got.dtype)
