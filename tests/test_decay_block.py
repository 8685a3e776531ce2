"""The block around decayed linear attention: training, prompts and single tokens give one answer (GPU), construction
and refusals (CPU)."""

import pytest
import torch

from nvsubquadratic_b200.decay_block import DecayBlockB200, DecayCache, DecayMixerB200
from nvsubquadratic_b200.sequence_mixer import QKVSequenceMixerB200
from oracle.decay_attention import decay_attention as attention_oracle
from oracle.layer_norm import layer_norm as norm_oracle
from oracle.rotary import rotary as rotary_oracle
from tests.conftest import rel_l2

gpu = pytest.mark.gpu


def test_construction():
    with pytest.raises(AssertionError, match="multiple of heads"):
        DecayMixerB200(100, 3)
    block = DecayBlockB200(64, 4).to(torch.bfloat16)
    assert block.norm.weight.dtype == torch.bfloat16
    assert block.mixer.mixer.log_decay.dtype == torch.float32  # decays keep their precision
    learned = DecayBlockB200(64, 4, learn_decay=True).to(torch.bfloat16)
    assert isinstance(learned.mixer.mixer.log_decay, torch.nn.Parameter)
    assert learned.mixer.mixer.log_decay.dtype == torch.float32
    assert DecayMixerB200(64, 4, rot_dim=0).turns is None
    cache = DecayCache(3, 2, 8)
    assert cache.rows(torch.tensor([2, -1, 3]), 3).tolist() == [2, 3, 3]
    with pytest.raises(AssertionError, match="as many slots"):
        cache.rows(None, 4)


def _reference(block, x):
    """The block in float64 from the oracles."""
    m, inner = block.mixer, block.mixer.mixer
    f = lambda t: t.detach().double().cpu()  # noqa: E731
    h = norm_oracle(x, block.norm.weight, block.norm.bias)
    qkv = h @ f(m.qkv_proj.weight).t()
    B, L, _ = x.shape
    q, k, v = qkv.view(B, L, 3, inner.heads, inner.head_dim).unbind(2)
    freq = f(inner.turns) / 2.0 ** 64 * 2 * torch.pi
    q, k = (rotary_oracle(t, freq, amplitude=inner.amplitude, interleaved=inner.interleaved) for t in (q, k))
    o, _ = attention_oracle(q, k, v, inner.log_decay)
    return f(x) + norm_oracle(o, eps=inner.eps).reshape(B, L, -1) @ f(m.out_proj.weight).t()


@gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_block_matches_the_oracle(interleaved):
    torch.manual_seed(0)
    block = DecayBlockB200(96, 3, interleaved=interleaved, rot_dim=20).cuda()
    x = torch.randn(2, 150, 96, device="cuda")
    # float32 throughout, the projections' sums of 96 terms included
    assert rel_l2(_reference(block, x), block(x)) <= 128 * 2.0 ** -24


@gpu
def test_training_step_reaches_every_parameter():
    torch.manual_seed(0)
    block = DecayBlockB200(128, 2, learn_decay=True).cuda()
    x = torch.randn(2, 70, 128, device="cuda", requires_grad=True)
    w = torch.randn(2, 70, 128, device="cuda")
    loss = (block(x) * w).sum()
    names = [n for n, _ in block.named_parameters()]
    grads = torch.autograd.grad(loss, [x, *block.parameters()])
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)
    # the decays' gradient against a central difference of the float64 reference along one direction
    i = 1 + names.index("mixer.mixer.log_decay")
    g = block.mixer.mixer.log_decay
    d, eps, ends = torch.tensor([1.0, -0.7], device="cuda"), 1e-3, []
    base = g.detach().clone()
    for sign in (1, -1):
        g.data = base + sign * eps * base * d
        ends.append((_reference(block, x) * w.double().cpu()).sum().item())
    g.data = base
    slope = (ends[0] - ends[1]) / (2 * eps)
    want = (grads[i] * base * d).sum().item()
    # truncation eps^2, and float32 forward and backward beside float64
    assert slope == pytest.approx(want, rel=1e-3, abs=1e-3 * abs(w).sum().item() ** 0.5)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_prompt_and_tokens_follow_the_sequence(dtype):
    torch.manual_seed(0)
    block = DecayBlockB200(128, 2).cuda().to(dtype)
    B, L, cuts = 3, 100, [37, 1, 80]
    x = torch.randn(B, L, 128, device="cuda", dtype=dtype)
    cache = DecayCache(5, 2, 64, device="cuda")
    cache.state.normal_()
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    cache.reset(slots)
    others = cache.state[[1, 3]].clone()
    tol = 256 * 2.0 ** -24 if dtype is torch.float32 else 0.02
    with torch.no_grad():
        want = block(x)
        padded = x.clone()
        for b, n in enumerate(cuts):
            padded[b, n:] = float("nan")
        y = block(padded[:, :max(cuts)], cache=cache, slots=slots,
                  lengths=torch.tensor(cuts, dtype=torch.int32, device="cuda"))
        for b, n in enumerate(cuts):
            assert rel_l2(want[b, :n], y[b, :n]) <= tol
        assert cache.position[slots.long()].tolist() == cuts
        for i in range(20):
            token = torch.stack([x[b, n + i] for b, n in enumerate(cuts)])[:, None]
            idle = slots.clone()
            if i == 7:
                idle[1] = -1  # one request waits
            y = block(token, cache=cache, slots=idle)
            for b, n in enumerate(cuts):
                if i < 7 or b != 1:
                    assert rel_l2(want[b, n + i], y[b, 0]) <= tol, (i, b)
        assert cache.position[slots.long()].tolist() == [57, 20, 100]
    assert torch.equal(cache.state[[1, 3]], others)


@gpu
def test_runs_in_the_qkv_mixer_and_refuses_context_parallel():
    mixer = DecayMixerB200(64, 1).cuda()
    layer = QKVSequenceMixerB200(64, mixer).cuda()
    assert layer(torch.randn(2, 4, 5, 64, device="cuda")).shape == (2, 4, 5, 64)  # a grid as a sequence of its points

    class Group:
        def size(self):
            return 2

    with pytest.raises(NotImplementedError, match="context-parallel"):
        layer(torch.randn(1, 4, 64, device="cuda"), Group())


@gpu
@pytest.mark.parametrize("lengths", [None, [9, 9, 4]], ids=["whole", "ragged"])
def test_idle_requests_of_a_prompt(lengths):
    """A slot outside the cache in a prompt call: zero mixer output whatever its tokens and earlier idle calls held, no state or
    position touched, and the same answer for the others."""
    torch.manual_seed(0)
    mixer = DecayMixerB200(64, 2).cuda()
    q, k, v = (torch.randn(3, 9, 64, device="cuda") for _ in range(3))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cache, want_cache = DecayCache(4, 2, 32, device="cuda"), DecayCache(4, 2, 32, device="cuda")
    with torch.no_grad():
        want = mixer(q, k, v, cache=want_cache, slots=torch.tensor([2, 0, 1], device="cuda"), lengths=n)
        bad = [t.clone() for t in (q, k, v)]
        for t in bad:
            t[1] = float("nan")
        slots = torch.tensor([2, 7, 1], device="cuda")
        for _ in range(2):  # what an idle request leaves behind must not matter to the next
            cache.reset(torch.tensor([1, 2], device="cuda"))
            got = mixer(*bad, cache=cache, slots=slots, lengths=n)
            assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and (got[1] == 0).all()
            slots[1] = -1
        assert torch.equal(cache.state[1:3], want_cache.state[1:3]) and (cache.state[[0, 3, 4]] == 0).all()
        assert cache.position.tolist() == [0, lengths[2] if lengths else 9, 9, 0, 0]
        token = mixer(*(t[:, :1] for t in bad), cache=cache, slots=slots)
        assert (token[1] == 0).all() and torch.isfinite(token).all() and (cache.state[[0, 3, 4]] == 0).all()
        assert cache.position.tolist() == [0, (lengths[2] if lengths else 9) + 1, 10, 0, 0]


def test_learned_decays_and_their_gradients_keep_their_precision():
    mixer = DecayMixerB200(64, 4, learn_decay=True)
    mixer.log_decay.grad = torch.randn(4)
    value, grad = mixer.log_decay.detach().clone(), mixer.log_decay.grad.clone()
    mixer.to(torch.bfloat16).half().double()
    assert mixer.log_decay.dtype == torch.float32 and torch.equal(mixer.log_decay, value)
    assert mixer.log_decay.grad.dtype == torch.float32 and torch.equal(mixer.log_decay.grad, grad)
    torch.optim.AdamW(mixer.parameters(), lr=0.1).step()
    assert not torch.equal(mixer.log_decay, value)


@gpu
def test_every_gradient_of_the_block():
    """x's and every parameter's gradient against torch's own differentiation of the block written out in float64. Five operators in
    a row, each good to 128 * 2^-24 of its result."""
    torch.manual_seed(0)
    B, L, C, H, rot = 2, 45, 96, 3, 20
    block = DecayBlockB200(C, H, learn_decay=True, rot_dim=rot, qkv_bias=True, out_proj_bias=True).cuda()
    with torch.no_grad():
        for p in block.parameters():
            if p is not block.mixer.mixer.log_decay:
                p.add_(0.1 * torch.randn_like(p))
    x, dy = torch.randn(B, L, C, device="cuda", requires_grad=True), torch.randn(B, L, C, device="cuda")
    names = ["x"] + [n for n, _ in block.named_parameters()]
    grads = torch.autograd.grad(block(x), [x, *block.parameters()], dy)

    P = {n: p.detach().double().cpu().requires_grad_() for n, p in block.named_parameters()}
    P["x"] = x.detach().double().cpu().requires_grad_()
    norm = torch.nn.functional.layer_norm
    h = norm(P["x"], (C,), P["norm.weight"], P["norm.bias"])
    qkv = (h @ P["mixer.qkv_proj.weight"].t() + P["mixer.qkv_proj.bias"]).view(B, L, 3, H, C // H)
    angle = torch.arange(L)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(t):
        a, b = t[..., :rot // 2], t[..., rot // 2:rot]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, t[..., rot:]), -1)

    q, k, v = turn(qkv[:, :, 0]), turn(qkv[:, :, 1]), qkv[:, :, 2]
    gap = torch.arange(L)[:, None] - torch.arange(L)
    weight = torch.exp(P["mixer.mixer.log_decay"][:, None, None] * gap.clamp(min=0)) * (gap >= 0)
    o = torch.einsum("bihd,bjhd,hij,bjhe->bihe", q, k, weight, v) * (C // H) ** -0.5
    y = P["x"] + norm(o, (C // H,)).reshape(B, L, C) @ P["mixer.out_proj.weight"].t() + P["mixer.out_proj.bias"]
    want = torch.autograd.grad(y, [P[n] for n in names], dy.double().cpu())
    bad = {n: rel_l2(w, g) for n, w, g in zip(names, want, grads) if not rel_l2(w, g) <= 5 * 128 * 2.0 ** -24}
    assert not bad, bad
