"""Log decays above 1: what the float32 recurrence holds comes out whatever the products of its decays are, on every number of rows.

Tolerance of an element, from the sizes M that the same recurrence has with every term taken positive: a decay of 16 or 32 bits is off
by 6 + 2 |gate| units of 2^-24 with its product and its sum (the exponential 4, its argument's rounding 1.5 |gate|, the product and the
sum 1 each), so a state after n tokens by n times that of M; a complement by 16 units more. A gate's gradient multiplies a state's
gradient with a state. 16-bit outputs are rounded once more. Numbers below 2^-126 have fewer digits: 2^-140 for all of their roundings.
"""

import pytest
import torch

from nvsubquadratic_b200.gated_scan import gated_scan
from oracle.gated_scan import gated_scan as oracle

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
UNIT = 2.0 ** -24
INF = float("inf")

# gates of the tokens, the initial state, the size of the inputs, the final state's gradient and the upstream gradients' size
CASES = {
    # a state that is small enough to grow through whole tiles, whose products pass 2^128
    "small states grow": ([0.75] * 150, 1e-20, 0.0, 1e-20, 0.0),
    "small inputs grow": ([0.75] * 150, 0.0, 1e-20, 0.0, 1e-20),
    "segments overflow": (([6.0] * 20 + [-6.0] * 20) * 4, 1e-27, 1e-30, 1e-27, 1e-30),
    # products that pass the smallest numbers and come back
    "shrinks, then grows": ([-1.5] * 64 + [1.5] * 64 + [-0.5] * 40, 1e10, 0.0, 1e-10, 0.0),
    "shrinks and grows in a segment": (([-12.0] * 8 + [12.0] * 8) * 9, 1e20, 1e-10, 1e-10, 1e-15),
    "grows, then shrinks": (([1.0] * 8 + [-1.0] * 8) * 16, 1.0, 0.0, 1.0, 0.0),
    "grows far, then shrinks": (([1.5] * 8 + [-1.5] * 8) * 16, 1.0, 1e-3, 1.0, 1e-3),
    # a decay of zero, then a product that overflows, and the other way round
    "forgets, then grows": ([-0.1] * 40 + [-INF] + [0.75] * 110, 1.0, 0.0, 1e-20, 0.0),
    "forgets, then overflows": ([-0.1] * 40 + [-INF] + [6.0] * 20 + [-0.5] * 70, 1.0, 0.0, 1e-25, 1e-30),
    "overflows, then forgets": ([6.0] * 20 + [-INF] + [0.25] * 100, 0.0, 0.0, 1e-3, 1e-30),
    # outputs and states far below what they come from, between a peak and a decay of zero
    "shrinks far, then forgets": (([5.0] * 10 + [0.0] * 6 + [-50.0] * 2 + [-INF] + [-0.1] * 13) * 4, 1e5, 0.0, 1e-5, 1e-5),
    "slow and fast": (([1e-3] * 30 + [-1e-3] * 30) * 4, 1.0, 1.0, 1.0, 1.0),
}
# copies of eight channels side by side: rows of 64 bytes that CTAs share, rows of 128 bytes that CTAs share, a CTA for each row
COPIES = {F32: {"few": 1, "some": 200, "many": 1250}, BF16: {"few": 1, "some": 400, "many": 2500}}
COPIES[F16] = COPIES[BF16]

# float16 where it holds the outputs
TYPED = [(n, d) for n in CASES for d in (F32, BF16, F16) if d is not F16 or n in ("grows, then shrinks", "slow and fast")]


def _case(name, dtype, seed=0):
    gates, h0, x, dstate, dy = CASES[name]
    g, L = torch.Generator().manual_seed(seed), len(gates)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(x=(x * r(1, L, 8)).to(dtype), gate=torch.tensor(gates)[None, :, None].expand(1, L, 8).to(dtype).contiguous(),
                initial_state=h0 * (1 + 0.1 * r(1, 8)), dy=(dy * r(1, L, 8)).to(dtype), dstate=dstate * (1 + 0.1 * r(1, 8)))


def _sizes(c, complement):
    """(outputs, final state, dx, dgate, dinitial_state), each with its tolerance for float32, in float64."""
    x, g, dy = (c[k].double() for k in ("x", "gate", "dy"))
    want = [t for t in oracle(c["x"], c["gate"], None, "log", complement, c["initial_state"], None, c["dy"], c["dstate"]) if t is not None]
    a, u = g.exp(), -torch.expm1(g)
    s = u.abs() if complement else torch.ones_like(u)
    L, unit = x.shape[1], (6 + 2 * g[g.isfinite()].abs().max().item() + 16) * UNIT
    M, h = [], c["initial_state"].double().abs()
    before = []
    for t in range(L):
        before.append(h)
        h = a[:, t] * h + s[:, t] * x[:, t].abs()
        M.append(h)
    M, before = torch.stack(M, 1), torch.stack(before, 1)
    G, w = torch.zeros_like(M), c["dstate"].double().abs()
    for t in range(L - 1, -1, -1):
        G[:, t] = dy[:, t].abs() + w
        w = a[:, t] * G[:, t]
    n = torch.arange(1, L + 1, dtype=torch.float64)[None, :, None] + 8
    floor = 2.0 ** -140
    tol = [unit * n * M + floor, unit * (L + 8) * M[:, -1] + floor,
           unit * (L + 10 - n + 8) * s * G + floor, None, unit * (L + 8) * w + floor]
    inner = before + x.abs() if complement else before
    tol[3] = 2 * unit * (L + 16) * a * G * inner + floor
    return want, tol


def test_the_cases_fit_float32():
    """Every value that is compared is one that float32 holds."""
    for name in CASES:
        for complement in (False, True):
            want, _ = _sizes(_case(name, F32), complement)
            assert all(t.abs().max() < 2.0 ** 126 for t in want), (name, [t.abs().max().item() for t in want])


@gpu
@pytest.mark.parametrize("copies", ["few", "some", "many"])
@pytest.mark.parametrize("name,dtype", TYPED, ids=[f"{n}-{str(d)[6:]}" for n, d in TYPED])
def test_products_out_of_range(name, dtype, copies):
    n = COPIES[dtype][copies]
    for complement in (False, True):
        c = _case(name, dtype)
        want, tol = _sizes(c, complement)
        wide = {k: t.repeat(*[1] * (t.ndim - 1), n).cuda() for k, t in c.items()}
        leaves = [wide[k].requires_grad_() for k in ("x", "gate", "initial_state")]
        y, state = gated_scan(leaves[0], leaves[1], form="log", complement=complement, initial_state=leaves[2], return_state=True)
        got = [y, state, *torch.autograd.grad([y, state], leaves, [wide["dy"], wide["dstate"]])]
        with torch.no_grad():
            again = gated_scan(wide["x"], wide["gate"], form="log", complement=complement, initial_state=wide["initial_state"],
                               return_state=True)
        assert torch.equal(again[0], y) and torch.equal(again[1], state)
        for i, (w, t, o) in enumerate(zip(want, tol, got)):
            o = o.detach().unflatten(-1, (n, 8))
            assert torch.equal(o, o[..., :1, :].expand_as(o)), i  # every copy of a channel has the same bits
            o = o[..., 0, :].double().cpu()
            least = 2.0 ** -25 if got[i].dtype is F16 else 2.0 ** -134 if got[i].dtype is BF16 else 2.0 ** -149
            held = torch.finfo(got[i].dtype).max
            err, allowed = (o - w).abs(), t + HALF_STEP[got[i].dtype] * (w.abs() + t) + least
            fine = w.abs() + t < held
            assert (err <= allowed)[fine].all(), (i, (err / allowed)[fine].max().item(), o.isfinite().all().item())


@gpu
@pytest.mark.parametrize("copies", ["few", "some", "many"])
def test_what_lies_beside_a_product_out_of_range(copies):
    """NaN and infinities in one channel, products out of range in another: each channel as if it were alone."""
    n, L = COPIES[F32][copies], 150
    g = torch.Generator().manual_seed(1)
    x, gate = torch.randn(1, L, 8, generator=g), -torch.rand(1, L, 8, generator=g)
    gate[..., 1], x[..., 1] = 0.75, 1e-20
    x[0, 60, 2], x[0, 70, 3] = float("nan"), INF
    gate[0, 80:, 3] = -8.0
    gate[..., 4], x[..., 4] = 3.0, 0.0
    want, end = oracle(x, gate, form="log", complement=False)
    y, state = gated_scan(x.repeat(1, 1, n).cuda(), gate.repeat(1, 1, n).cuda(), form="log", complement=False, return_state=True)
    for w, o in ((want, y), (end, state)):
        o = o.unflatten(-1, (n, 8))[..., 0, :].double().cpu()
        assert torch.equal(w.isnan(), o.isnan()) and torch.equal(w.isinf(), o.isinf())
        fine = w.isfinite()
        # 150 tokens of 8 units, states of terms of either sign that a bound of 10 times their size covers
        assert ((o - w).abs() <= 150 * 8 * UNIT * (w.abs() + 10))[fine].all()
        ch = o[..., 1] / w[..., 1]
        assert ((ch - 1).abs() <= 150 * 8 * UNIT).all()
        assert (o[..., 4] == 0).all()
