"""The gated block, its cache, and the decayed attention's mixer with normed queries and keys: training, prompts, single tokens,
forked and compacted requests give one answer (GPU), construction and refusals (CPU)."""

import pytest
import torch

from nvsubquadratic_b200.decay_block import DecayBlockB200, DecayCache, DecayMixerB200
from nvsubquadratic_b200.gated_block import GatedBlockB200, GatedCache, GatedMixerB200
from nvsubquadratic_b200.sequence_mixer import QKVSequenceMixerB200
from oracle.decay_attention import decay_attention as attention_oracle
from oracle.decay_attention import decay_attention_grads as attention_grads
from oracle.gated_scan import gated_scan as scan_oracle
from oracle.layer_norm import layer_norm as norm_oracle
from oracle.qk_norm import qk_norm_rotary as qk_oracle
from oracle.rotary import rotary as rotary_oracle
from tests.conftest import rel_l2

gpu = pytest.mark.gpu


def test_construction():
    block = GatedBlockB200(64)
    keep = torch.sigmoid(block.mixer.qkv_proj.bias[64:128])
    assert keep[0].item() == pytest.approx(1 - 1 / 16) and keep[-1].item() == pytest.approx(1 - 1 / 4096, abs=1e-6)
    cache = GatedCache(3, 8)
    assert cache.rows(torch.tensor([2, -1, 3]), 3).tolist() == [2, 3, 3] and cache.pools()[0].shape == (3, 8)
    with pytest.raises(AssertionError, match="as many slots"):
        cache.rows(None, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.fork(torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    plain, normed = DecayMixerB200(64, 4), DecayMixerB200(64, 4, qk_norm=True)
    assert set(plain.state_dict()) == {"log_decay"}  # as before
    assert set(normed.state_dict()) == {"log_decay", "q_norm", "k_norm"} and normed.q_norm.shape == (16,)


def _reference(block, x):
    """The gated block in float64 from the oracles."""
    m = block.mixer
    f = lambda t: t.detach().double().cpu()  # noqa: E731
    h = norm_oracle(x, block.norm.weight, block.norm.bias)
    q, k, v = (h @ f(m.qkv_proj.weight).t() + f(m.qkv_proj.bias)).chunk(3, -1)
    y, _ = scan_oracle(v, k, q)
    return f(x) + y @ f(m.out_proj.weight).t()


@gpu
def test_block_matches_the_oracle():
    torch.manual_seed(0)
    block = GatedBlockB200(96).cuda()
    x = torch.randn(2, 150, 96, device="cuda")
    # float32 throughout, the projections' sums of 96 terms included
    assert rel_l2(_reference(block, x), block(x)) <= 128 * 2.0 ** -24


@gpu
def test_every_gradient_of_the_block():
    """x's and every parameter's gradient against torch's own differentiation of the block written out in float64. Four operators in a
    row, each good to 128 * 2^-24 of its result."""
    torch.manual_seed(0)
    B, L, C = 2, 45, 32
    block = GatedBlockB200(C, out_proj_bias=True).cuda()
    with torch.no_grad():
        for p in block.parameters():
            p.add_(0.1 * torch.randn_like(p))
    x, dy = torch.randn(B, L, C, device="cuda", requires_grad=True), torch.randn(B, L, C, device="cuda")
    names = ["x"] + [n for n, _ in block.named_parameters()]
    grads = torch.autograd.grad(block(x), [x, *block.parameters()], dy)
    P = {n: p.detach().double().cpu().requires_grad_() for n, p in block.named_parameters()}
    P["x"] = x.detach().double().cpu().requires_grad_()
    h = torch.nn.functional.layer_norm(P["x"], (C,), P["norm.weight"], P["norm.bias"])
    q, k, v = (h @ P["mixer.qkv_proj.weight"].t() + P["mixer.qkv_proj.bias"]).chunk(3, -1)
    a, s, out = torch.sigmoid(k), torch.zeros(B, C, dtype=torch.float64), []
    for t in range(L):
        s = a[:, t] * s + (1 - a[:, t]) * v[:, t]
        out.append(s * torch.nn.functional.silu(q[:, t]))
    y = P["x"] + torch.stack(out, 1) @ P["mixer.out_proj.weight"].t() + P["mixer.out_proj.bias"]
    want = torch.autograd.grad(y, [P[n] for n in names], dy.double().cpu())
    bad = {n: rel_l2(w, g) for n, w, g in zip(names, want, grads) if not rel_l2(w, g) <= 4 * 128 * 2.0 ** -24}
    assert not bad, bad


def _blocks():
    return [("gated", lambda: GatedBlockB200(128), lambda n: GatedCache(n, 128, device="cuda")),
            ("decay", lambda: DecayBlockB200(128, 2, qk_norm=True, rot_dim=40), lambda n: DecayCache(n, 2, 64, device="cuda"))]


@gpu
@pytest.mark.parametrize("kind,make,hold", _blocks(), ids=[b[0] for b in _blocks()])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_serving_follows_the_sequence(kind, make, hold, dtype):
    """Prompts of unequal length, each answered twice from a fork, single tokens with one request idle, requests that end and the rest
    moved together: every output is the sequence's own."""
    torch.manual_seed(0)
    block, cache = make().cuda().to(dtype), hold(7)
    B, L, cuts = 3, 60, [20, 1, 33]
    x = torch.randn(2 * B, L, 128, device="cuda", dtype=dtype)
    x[B:] = torch.where(torch.arange(L, device="cuda")[None, :, None] < torch.tensor(cuts, device="cuda")[:, None, None], x[:B], x[B:])
    tol = 256 * 2.0 ** -24 if dtype is torch.float32 else 0.02
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for t in cache.tensors():
        t.fill_(3)
    slots = [4, 0, 2, 6, 1, 5]  # of the six sequences; slot 3 is nobody's
    cache.reset(i32(slots[:B]))
    other = [t[3].clone() for t in cache.tensors()]
    with torch.no_grad():
        want = block(x)
        padded = x[:B].clone()
        for b, n in enumerate(cuts):
            padded[b, n:] = float("nan")
        y = block(padded[:, :max(cuts)], cache=cache, slots=i32(slots[:B]), lengths=i32(cuts))
        for b, n in enumerate(cuts):
            assert rel_l2(want[b, :n], y[b, :n]) <= tol
        cache.fork(i32(slots[:B]), i32(slots[B:]))
        at = cuts * 2

        def token(who, where):
            y = block(torch.stack([x[b, at[b]] for b in who])[:, None], cache=cache, slots=i32(where))
            for i, b in enumerate(who):
                if 0 <= where[i] < 7:
                    assert rel_l2(want[b, at[b]], y[i, 0]) <= tol, b
                    at[b] += 1

        for _ in range(5):
            token(range(6), slots)
        token(range(6), [*slots[:2], -1, *slots[3:]])  # one waits
        assert all(torch.equal(t[3], o) for t, o in zip(cache.tensors(), other))
        stay = [0, 2, 3, 5]
        live = torch.zeros(7, dtype=torch.bool, device="cuda")
        live[[slots[b] for b in stay]] = True
        moved = cache.compact(live).tolist()
        where = [moved[slots[b]] for b in stay]
        assert sorted(where) == [0, 1, 2, 3]
        for _ in range(5):
            token(stay, where)


@gpu
@pytest.mark.parametrize("lengths", [None, [9, 9, 4]], ids=["whole", "ragged"])
def test_idle_requests_of_a_prompt(lengths):
    torch.manual_seed(0)
    mixer, cache, want_cache = GatedMixerB200(), GatedCache(4, 64, device="cuda"), GatedCache(4, 64, device="cuda")
    q, k, v = (torch.randn(3, 9, 64, device="cuda") for _ in range(3))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = mixer(q, k, v, cache=want_cache, slots=torch.tensor([2, 0, 1], device="cuda"), lengths=n)
    bad = [t.clone() for t in (q, k, v)]
    for t in bad:
        t[1] = float("nan")
    for idle in (7, -1):
        cache.reset(torch.tensor([1, 2], device="cuda"))
        got = mixer(*bad, cache=cache, slots=torch.tensor([2, idle, 1], device="cuda"), lengths=n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and (got[1] == 0).all()
    assert torch.equal(cache.state[1:3], want_cache.state[1:3]) and (cache.state[[0, 3, 4]] == 0).all()
    one = mixer(*(t[:, :1] for t in bad), cache=cache, slots=torch.tensor([2, -1, 1], device="cuda"))
    assert (one[1] == 0).all() and torch.isfinite(one).all() and (cache.state[[0, 3, 4]] == 0).all()


@gpu
def test_grids_and_context_parallel_groups():
    layer = QKVSequenceMixerB200(64, GatedMixerB200()).cuda()
    assert layer(torch.randn(2, 4, 5, 64, device="cuda")).shape == (2, 4, 5, 64)  # a grid as a sequence of its points

    class Group:
        def size(self):
            return 2

    with pytest.raises(NotImplementedError, match="context-parallel"):
        layer(torch.randn(1, 4, 64, device="cuda"), Group())


@gpu
@pytest.mark.parametrize("rot_dim", [None, 0, 20])
def test_decay_mixer_with_normed_queries_and_keys(rot_dim):
    torch.manual_seed(0)
    mixer = DecayMixerB200(96, 3, rot_dim=rot_dim, qk_norm=True).cuda()
    with torch.no_grad():
        mixer.q_norm.add_(0.2 * torch.randn_like(mixer.q_norm)), mixer.k_norm.add_(0.2 * torch.randn_like(mixer.k_norm))
    q, k, v = (torch.randn(2, 70, 96, device="cuda") for _ in range(3))
    heads = lambda t: t.unflatten(-1, (3, 32))  # noqa: E731
    freq = None if mixer.turns is None else mixer.turns.double().cpu() / 2.0 ** 64 * 2 * torch.pi
    a, b = (qk_oracle(heads(t), w, freq) for t, w in ((q, mixer.q_norm), (k, mixer.k_norm)))
    want = norm_oracle(attention_oracle(a, b, heads(v), mixer.log_decay)[0], eps=mixer.eps).reshape(2, 70, 96)
    out = mixer(q, k, v)
    assert rel_l2(want, out) <= 256 * 2.0 ** -24
    grads = torch.autograd.grad((out * torch.randn_like(out)).sum(), [mixer.q_norm, mixer.k_norm])
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)


@gpu
def test_any_number_of_slots_is_reset():
    """More slots than one call of copy_slots takes; slots outside the cache, past 32 bits too, clear nothing."""
    cache = GatedCache(20001, 4, device="cuda")
    cache.state.fill_(3)
    cache.reset(torch.arange(20000, device="cuda"))
    assert (cache.state[:20000] == 0).all() and (cache.state[20000:] == 3).all()
    cache.state.fill_(3)
    cache.reset(torch.tensor([-1, 5, 20001, 1 << 32, (1 << 32) + 7], device="cuda"))
    assert (cache.state[5] == 0).all() and cache.state.sum().item() == 3 * 4 * 20001
    cache.reset(torch.zeros(0, dtype=torch.int64, device="cuda"))


@gpu
def test_gradients_of_the_norms_of_queries_and_keys():
    """Through the decayed mixer, against the oracles' formulas one after the other. A weight's gradient is a sum of n terms, (n + 128)
    units of their sizes, and what comes to it has gone through the layer norm's and the attention's, 256 units each way."""
    torch.manual_seed(0)
    B, L, H, D = 2, 70, 3, 32
    mixer = DecayMixerB200(H * D, H, rot_dim=20, qk_norm=True).cuda()
    with torch.no_grad():
        mixer.q_norm.add_(0.2 * torch.randn_like(mixer.q_norm)), mixer.k_norm.add_(0.2 * torch.randn_like(mixer.k_norm))
    q, k, v, dy = (torch.randn(B, L, H * D, device="cuda") for _ in range(4))
    grads = torch.autograd.grad(mixer(q, k, v), [mixer.q_norm, mixer.k_norm], dy)
    q, k, v, dy = (t.cpu().unflatten(-1, (H, D)) for t in (q, k, v, dy))
    freq = mixer.turns.double().cpu() / 2.0 ** 64 * 2 * torch.pi
    a, b = qk_oracle(q, mixer.q_norm, freq), qk_oracle(k, mixer.k_norm, freq)
    o, _ = attention_oracle(a, b, v, mixer.log_decay)
    do = norm_oracle(o, eps=mixer.eps, dy=dy)[1]
    ups = attention_grads(a, b, v, mixer.log_decay, do)[:2]
    for x, w, up, got in zip((q, k), (mixer.q_norm, mixer.k_norm), ups, grads):
        want = qk_oracle(x, w, freq, dy=up)[2]
        h = x.double() / x.double().square().mean(-1, keepdim=True).add(1e-6).sqrt()
        sizes = (rotary_oracle(up, freq, backward=True) * h).abs().sum((0, 1, 2))
        assert (want - got.double().cpu()).norm() <= (B * L * H + 128 + 4 * 256) * 2.0 ** -24 * sizes.norm()


@gpu
@pytest.mark.parametrize("kind,make,hold", _blocks(), ids=[b[0] for b in _blocks()])
def test_training_on_ragged_sequences(kind, make, hold):
    """A padded batch gives the gradients of its sequences one by one; padding passes the residual on and nothing else. Either side is good
    to four operators of 128 units each."""
    torch.manual_seed(0)
    block, lengths = make().cuda(), [90, 0, 33, 1]
    x, dy = (torch.randn(4, 90, 128, device="cuda") for _ in range(2))
    for b, n in enumerate(lengths):
        dy[b, n:] = 0
    leaves = [x.requires_grad_(), *block.parameters()]
    y = block(x, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    got = torch.autograd.grad(y, leaves, dy)
    want = [torch.zeros_like(t, dtype=torch.float64) for t in leaves]
    for b, n in enumerate(lengths):
        assert torch.equal(y[b, n:], x[b, n:])
        if n:
            alone = block(x[b:b + 1, :n])
            assert rel_l2(alone[0], y[b, :n]) <= 256 * 2.0 ** -24
            for w, g in zip(want, torch.autograd.grad(alone, leaves, dy[b:b + 1, :n])):
                w += g
    bad = [(i, rel_l2(w, g)) for i, (w, g) in enumerate(zip(want, got)) if not rel_l2(w, g) <= 2 * 4 * 128 * 2.0 ** -24]
    assert not bad, bad


class _PlainScan(torch.nn.Module):
    """The gated mixer in float64, rounded where GatedMixerB200 rounds."""

    def forward(self, query, key, value, cp_group=None, **kw):
        a, u, s, out = torch.sigmoid(key.double()), torch.sigmoid(-key.double()), 0, []
        for t in range(key.shape[1]):
            s = a[:, t] * s + u[:, t] * value[:, t].double()
            out.append(s)
        return (torch.stack(out, 1) * torch.nn.functional.silu(query.double())).to(value.dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_16_bit_gradients_of_the_block(dtype):
    """Against the same block with the scan written out. Both round the scan's output and its three gradients, to the same or to
    neighbouring numbers: four times a step, 2 eps / 2 each."""
    torch.manual_seed(0)
    block = GatedBlockB200(64).cuda().to(dtype)
    x, dy = (torch.randn(2, 40, 64, device="cuda", dtype=dtype) for _ in range(2))
    leaves = [x.requires_grad_(), *block.parameters()]
    got = torch.autograd.grad(block(x), leaves, dy)
    block.mixer.mixer = _PlainScan()
    want = torch.autograd.grad(block(x), leaves, dy)
    bad = [(i, rel_l2(w, g)) for i, (w, g) in enumerate(zip(want, got)) if not rel_l2(w, g) <= 4 * torch.finfo(dtype).eps]
    assert not bad, bad
