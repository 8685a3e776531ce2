"""Measured calls of the decayed linear attention mixer and of what stands around it in a block:

* ``attention`` — linear attention with one decay for each head over whole sequences
  (``decay_attention``), forward for prompts, forward and backward for training;
* ``step`` — the same operator's recurrent form for one token of every running sequence
  (``decay_attention_step``);
* ``rotary`` — rotary positions of queries and keys (``rotary``), forward for serving, forward and
  backward for training;
* ``norm`` — layer norm over the last axis (``layer_norm``), forward for serving, forward and
  backward with the weight and bias gradients for training.

The sizes are those of the mixers this package benchmarks (a 14 x 14 grid of 768 channels, a
128 x 128 grid of 256 channels, long sequences of up to 4096 channels), taken as sequences with
heads of 64 or 128 channels, and odd ones between them. ``run`` calls the package where ``own`` is
true; elsewhere it computes the same outputs from elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one sequence being answered, the 768-channel mixer: nothing but latency
        dict(name="step_one", op="step", dtype="bf16", B=1, H=12, Hk=12, Dk=64, Dv=64, pool=0),
        # a serving step of 200 requests in a pool of 224 slots at 4096 channels, some slots idle
        dict(name="step_pool", op="step", dtype="bf16", B=200, H=32, Hk=32, Dk=128, Dv=128, pool=224),
        # prompts of unequal length in one batch, three query heads sharing each key/value head
        dict(name="prompt_ragged", op="attention", dtype="bf16", B=16, L=1023, H=12, Hk=4, Dk=64, Dv=64,
             ragged=True, start=True, train=False, learn=False),
        # one long prompt: 8 rows only, so the long axis has to feed the machine
        dict(name="prompt_long", op="attention", dtype="bf16", B=1, L=65536, H=8, Hk=8, Dk=128, Dv=128,
             ragged=False, start=False, train=False, learn=False),
        # training on the 128 x 128 grid of 256 channels as a sequence
        dict(name="train_grid", op="attention", dtype="bf16", B=8, L=16384, H=4, Hk=4, Dk=64, Dv=64,
             ragged=False, start=False, train=True, learn=False),
        # a small 32-bit run with learned decays, an initial state, odd lengths and head sizes
        dict(name="train_f32_odd", op="attention", dtype="f32", B=2, L=1001, H=6, Hk=3, Dk=40, Dv=72,
             ragged=True, start=True, train=True, learn=True),
        # the queries and keys of one token of 32 requests at unequal positions
        dict(name="rotary_token", op="rotary", dtype="bf16", B=32, L=1, H=12, Hk=4, D=64, rot=64, interleaved=False,
             scaling="none", positions="each", train=False),
        # training on a long sequence of 4096 channels, positions stretched for long contexts
        dict(name="rotary_train", op="rotary", dtype="bf16", B=1, L=65536, H=32, Hk=32, D=128, rot=128,
             interleaved=False, scaling="ramp", positions="none", train=True),
        # neighbouring pairs, 50 of 80 features turned, odd lengths, half precision
        dict(name="rotary_part", op="rotary", dtype="f16", B=3, L=1021, H=5, Hk=5, D=80, rot=50, interleaved=True,
             scaling="linear", positions="each", train=True),
        # one token of 32 requests, 768 channels
        dict(name="norm_token", op="norm", dtype="bf16", rows=32, C=768, affine=True, train=False),
        # training on a long sequence of 4096 channels
        dict(name="norm_train", op="norm", dtype="bf16", rows=65536, C=4096, affine=True, train=True),
        # odd rows and channels in 32 bits
        dict(name="norm_f32_odd", op="norm", dtype="f32", rows=6271, C=771, affine=True, train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["step", "attention", "attention", "attention", "rotary", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        C = _log_int(rng, 33, 4096)
        rows = _log_int(rng, 1, min(65536, (1 << 27) // C))
        return dict(op=op, dtype=dtype, rows=rows, C=C, affine=rng.random() < 0.8, train=rng.random() < 0.6)
    Hk = rng.choice([1, 2, 4, 6, 8])
    H = Hk * rng.choice([1, 1, 2, 3])
    B = _log_int(rng, 1, 32)
    if op == "rotary":
        D = rng.choice([64, 128, 80, rng.randrange(16, 257)])
        rot = max(2, min(D, rng.choice([D, D // 2, rng.randrange(2, D + 1)])) // 2 * 2)
        L = _log_int(rng, 1, max(1, min(65536, (1 << 26) // (B * H * D))))
        return dict(op=op, dtype=dtype, B=B, L=L, H=H, Hk=Hk, D=D, rot=rot, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "ramp"]), positions=rng.choice(["none", "each"]),
                    train=rng.random() < 0.5)
    Dk = rng.choice([64, 64, 128, rng.randrange(8, 129)])
    Dv = rng.choice([Dk, Dk, 64, rng.randrange(8, 129)])
    if op == "step":
        B = _log_int(rng, 1, max(1, min(512, (1 << 26) // (H * Dk * Dv))))
        return dict(op=op, dtype=dtype, B=B, H=H, Hk=Hk, Dk=Dk, Dv=Dv, pool=rng.choice([0, B + 3]))
    train = rng.random() < 0.5
    most = (1 << 22 if dtype == "f32" else 1 << 24) // (B * H * max(Dk, Dv))
    L = _log_int(rng, 1, max(1, min(32768, most)))
    return dict(op=op, dtype=dtype, B=B, L=L, H=H, Hk=Hk, Dk=Dk, Dv=Dv, ragged=rng.random() < 0.4,
                start=rng.random() < 0.4, train=train, learn=train and L <= 2048 and rng.random() < 0.3)


# ---------------------------------------------------------------- inputs


def _randn(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _log_decay(H):
    """Horizons from 16 tokens to 4096, one for each head."""
    horizon = 2.0 ** torch.linspace(4.0, 12.0, H, dtype=torch.float64)
    return torch.log1p(-1.0 / horizon).to(device="cuda", dtype=torch.float32)


def _frequencies(case):
    """Angle per position of each pair, and the amplitude, from the definition."""
    rot, base = case["rot"], 10000.0
    if case["scaling"] == "ntk":
        base = base * 4.0 ** (rot / max(rot - 2, 1))
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    freq = base ** (-2.0 * i / rot)
    amp = 1.0
    if case["scaling"] == "linear":
        freq = freq / 4.0
    elif case["scaling"] == "ramp":
        # pairs that turn more than 32 times over the 8192 positions keep their frequency, those
        # that turn less than once are slowed by 8, those between are blended by their index
        lo = rot * math.log(8192 / (32 * 2 * math.pi)) / (2 * math.log(base))
        hi = rot * math.log(8192 / (1 * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot // 2 - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        freq = freq / 8.0 * (1 - keep) + freq * keep
        amp = 0.1 * math.log(8.0) + 1.0
    return freq, amp


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        rows, C = case["rows"], case["C"]
        s["x"] = (_randn(gen, (rows, C)) * 1.5 + 0.3).to(dt)
        s["weight"] = (1 + 0.2 * _randn(gen, (C,))).to(dt) if case["affine"] else None
        s["bias"] = (0.1 * _randn(gen, (C,))).to(dt) if case["affine"] else None
        if case["train"]:
            s["dy"] = _randn(gen, (rows, C), dt)
        return s
    B, H, Hk = case["B"], case["H"], case["Hk"]
    if case["op"] == "rotary":
        L, D = case["L"], case["D"]
        s["q"], s["k"] = _randn(gen, (B, L, H, D), dt), _randn(gen, (B, L, Hk, D), dt)
        s["positions"] = None
        if case["positions"] == "each":  # each request goes on from where its cache ends
            s["positions"] = (torch.randint(0, 100000, (B, 1), generator=gen, device="cuda")
                              + torch.arange(L, device="cuda"))
        if case["train"]:
            s["dq"], s["dk"] = _randn(gen, (B, L, H, D), dt), _randn(gen, (B, L, Hk, D), dt)
        # turns per position in units of 2^-64, so that whole turns drop out exactly
        freq, s["amplitude"] = _frequencies(case)
        s["turns"] = torch.tensor([int(f / (2 * math.pi) * 2.0 ** 64) for f in freq.tolist()], device="cuda")
        return s
    Dk, Dv = case["Dk"], case["Dv"]
    s["log_decay"] = _log_decay(H)
    if case["op"] == "step":
        N = case["pool"] or B
        s["q"], s["k"], s["v"] = _randn(gen, (B, H, Dk), dt), _randn(gen, (B, Hk, Dk), dt), _randn(gen, (B, Hk, Dv), dt)
        s["state"] = 4 * _randn(gen, (N, H, Dk, Dv))
        s["new_state"] = s["state"].clone()
        s["slots"] = None
        if case["pool"]:  # every seventh request has no slot and is passed over
            s["slots"] = torch.randperm(N, generator=gen, device="cuda")[:B].to(torch.int32)
            s["slots"][5::7] = -1
        return s
    L = case["L"]
    s["q"], s["k"], s["v"] = (_randn(gen, (B, L, H, Dk), dt), _randn(gen, (B, L, Hk, Dk), dt),
                              _randn(gen, (B, L, Hk, Dv), dt))
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, L + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        s["lengths"][0] = L
        s["lengths"][1:2] = 0
        s["lengths"][2:3] = 1
    s["initial_state"] = 2 * _randn(gen, (B, H, Dk, Dv)) if case["start"] else None
    if case["train"]:
        s["do"] = _randn(gen, (B, L, H, Dv), dt)
    return s


# ---------------------------------------------------------------- the plain forms, 32 bits


def _plain_attention(q, k, v, log_decay, S0, lengths):
    """The chunked form: products inside chunks of 128 tokens, and between them the chunks' states."""
    B, L, H, Dk = q.shape
    Dv, C = v.shape[-1], 128
    n = -(-L // C)
    scale = Dk ** -0.5
    t = torch.arange(L, device=q.device)
    live = t < lengths[:, None] if lengths is not None else torch.ones(B, L, dtype=torch.bool, device=q.device)
    live = live[:, :, None, None]

    def lay(x, heads):  # [B, L, h, D] -> [B, H, n, C, D], nothing past the length
        x = torch.where(live, x.float(), 0.0).repeat_interleave(H // heads, dim=2)
        return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * C - L)).view(B, n, C, H, -1).permute(0, 3, 1, 2, 4)

    Q, K, V = lay(q, q.shape[2]) * scale, lay(k, k.shape[2]), lay(v, v.shape[2])
    g = log_decay.float()
    i = torch.arange(C, device=q.device)
    gap = i[:, None] - i[None, :]
    inside = torch.exp(g[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
    o = (Q @ K.transpose(-1, -2) * inside[None, :, None]) @ V
    local = (K * torch.exp(g[:, None] * (C - 1 - i))[None, :, None, :, None]).transpose(-1, -2) @ V
    m = torch.arange(n, device=q.device)
    hop = m[:, None] - 1 - m[None, :]
    between = torch.exp(g[:, None, None] * C * hop.clamp(min=0)) * (hop >= 0)
    before = (between @ local.reshape(B, H, n, Dk * Dv)).view(B, H, n, Dk, Dv)
    if S0 is not None:
        before = before + torch.exp(g[:, None] * C * m)[None, :, :, None, None] * S0[:, :, None]
    o = o + (Q * torch.exp(g[:, None] * (i + 1))[None, :, None, :, None]) @ before
    o = torch.where(live, o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, Dv)[:, :L], 0.0)
    ends = lengths if lengths is not None else torch.full((B,), L, device=q.device)
    left = ends[:, None] - 1 - torch.arange(n * C, device=q.device)
    w = torch.exp(g[None, :, None] * left[:, None].clamp(min=0)) * (left >= 0)[:, None]
    state = (K.reshape(B, H, n * C, Dk) * w[..., None]).transpose(-1, -2) @ V.reshape(B, H, n * C, Dv)
    if S0 is not None:
        state = state + torch.exp(g[None] * ends[:, None])[..., None, None] * S0
    return o.to(q.dtype), state


def _plain_step(s):
    q, k, v, state, slots = s["q"], s["k"], s["v"], s["state"], s["slots"]
    H, Dk = q.shape[1:]
    at = slots.long().clamp(min=0) if slots is not None else torch.arange(q.shape[0], device=q.device)
    on = (slots >= 0) if slots is not None else torch.ones_like(at, dtype=torch.bool)
    K = k.float().repeat_interleave(H // k.shape[1], dim=1)
    V = v.float().repeat_interleave(H // v.shape[1], dim=1)
    new = torch.exp(s["log_decay"])[None, :, None, None] * state[at] + K[..., :, None] * V[..., None, :]
    o = ((q.float() * Dk ** -0.5)[..., None] * new).sum(-2)
    s["new_state"][at[on]] = new[on]
    return torch.where(on[:, None, None], o, 0.0).to(q.dtype), s["new_state"]


def _plain_turn(x, cos, sin, rot, interleaved):
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(s):
    case, q, k = s["case"], s["q"], s["k"]
    p = s["positions"] if s["positions"] is not None else torch.arange(q.shape[1], device=q.device)[None]
    part = (p[..., None] * s["turns"]) >> 32  # 64-bit products wrap: what is left is the turn's fraction
    angle = part.float() * (2 * math.pi / 2.0 ** 32)
    cos, sin = (angle.cos() * s["amplitude"])[:, :, None], (angle.sin() * s["amplitude"])[:, :, None]
    rot, inter = case["rot"], case["interleaved"]
    out = [_plain_turn(q, cos, sin, rot, inter).to(q.dtype), _plain_turn(k, cos, sin, rot, inter).to(k.dtype)]
    if case["train"]:  # a turn's transpose is the turn back
        out += [_plain_turn(s["dq"], cos, -sin, rot, inter).to(q.dtype),
                _plain_turn(s["dk"], cos, -sin, rot, inter).to(k.dtype)]
    return out


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    h = c * rstd
    y = h if w is None else h * w.float() + b.float()
    out = [y.to(s["x"].dtype)]
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy if w is None else dy * w.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        out.append(dx.to(s["x"].dtype))
        if w is not None:
            out += [(dy * h).sum(0).to(w.dtype), dy.sum(0).to(b.dtype)]
    return out


# ---------------------------------------------------------------- one pass


def _attention(s, call):
    case = s["case"]
    names = ["q", "k", "v"] + (["initial_state"] if case["start"] else []) + (["log_decay"] if case["learn"] else [])
    given = dict(s)
    if case["train"]:
        given.update({n: s[n].detach().requires_grad_() for n in names})
    o, state = call(given)
    if not case["train"]:
        return [o, state]
    return [o, state, *torch.autograd.grad(o, [given[n] for n in names], s["do"])]


def _own(s):
    case = s["case"]
    if case["op"] == "step":
        from nvsubquadratic_b200.decay_attention import decay_attention_step

        o = decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"],
                                 out_state=s["new_state"])
        return [o, s["new_state"]]
    if case["op"] == "attention":
        from nvsubquadratic_b200.decay_attention import decay_attention

        return _attention(s, lambda a: decay_attention(a["q"], a["k"], a["v"], a["log_decay"], lengths=a["lengths"],
                                                       initial_state=a["initial_state"], return_state=True))
    if case["op"] == "rotary":
        from nvsubquadratic_b200.rotary import rotary

        q, k = s["q"], s["k"]
        if case["train"]:
            q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = rotary(q, k, s["turns"], positions=s["positions"], amplitude=s["amplitude"],
                     interleaved=case["interleaved"])
        if case["train"]:
            return [*out, *torch.autograd.grad(out, [q, k], [s["dq"], s["dk"]])]
        return list(out)
    from nvsubquadratic_b200.layer_norm import layer_norm

    args = [s["x"], s["weight"], s["bias"]]
    if not case["train"]:
        return [layer_norm(*args)]
    args = [a.detach().requires_grad_() if a is not None else None for a in args]
    y = layer_norm(*args)
    return [y, *torch.autograd.grad(y, [a for a in args if a is not None], s["dy"])]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "step":
        return list(_plain_step(state))
    if op == "attention":
        return _attention(state, lambda a: _plain_attention(a["q"], a["k"], a["v"], a["log_decay"], a["initial_state"],
                                                            a["lengths"]))
    return _plain_rotary(state) if op == "rotary" else _plain_norm(state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    passes = 2 if case.get("train") else 1
    if case["op"] == "norm":
        n, C = case["rows"] * case["C"], case["C"] * (2 if case["affine"] else 0)
        # x and y; dy and dx
        return {"bytes": e * (2 * n * passes + C * passes), "flops": 8 * n + (14 * n if case["train"] else 0)}
    B, H, Hk = case["B"], case["H"], case["Hk"]
    if case["op"] == "rotary":
        n = B * case["L"] * (H + Hk)
        places = 8 * B * case["L"] if case["positions"] == "each" else 0
        return {"bytes": 2 * e * n * case["D"] * passes + places, "flops": 3 * n * case["rot"] * passes}
    Dk, Dv = case["Dk"], case["Dv"]
    if case["op"] == "step":
        on = B - (len(range(5, B, 7)) if case["pool"] else 0)
        return {"bytes": 8 * on * H * Dk * Dv + e * B * (H + Hk) * (Dk + Dv) + 4 * H + (4 * B if case["pool"] else 0),
                "flops": 5 * on * H * Dk * Dv}
    L = case["L"]
    # ragged lengths are uniform over 0..L: the first is L, the second 0, the third 1
    tokens = B * L
    if case["ragged"]:
        tokens = L + (1 if B > 2 else 0) + max(0, B - 3) * L // 2
    out = B * L * H * Dv  # zeros are written past the lengths too
    read = tokens * (H * Dk + Hk * (Dk + Dv))
    states = 4 * B * H * Dk * Dv
    byts = e * (read + out) + states * (2 if case["start"] else 1) + 4 * H
    flops = 4 * tokens * H * Dk * Dv
    if case["train"]:
        byts += e * (tokens * H * Dv + B * L * (H * Dk + Hk * (Dk + Dv))) + (states if case["start"] else 0)
        flops += 8 * tokens * H * Dk * Dv + (4 * tokens * H * Dk * Dv if case["learn"] else 0)
    return {"bytes": byts, "flops": flops}


# ---------------------------------------------------------------- 64 bits, from the definitions


def _exact_attention(case, s):
    """The recurrence, token by token: S_t = a S_{t-1} + k_t v_t^T, o_t = S_t^T q_t / sqrt(Dk), and for the
    decay's gradient its derivative T_t = dS_t / dlog(a) = a (T_{t-1} + S_{t-1}); backwards in time
    G_t = a G_{t+1} + q_t do_t^T / sqrt(Dk), dk_t = G_t v_t, dv_t = G_t^T k_t."""
    B, L, H, Hk, Dk, Dv = (case[n] for n in ("B", "L", "H", "Hk", "Dk", "Dv"))
    r = H // Hk
    if 3 * 8 * B * H * Dk * Dv > 4e9 or L * (6e-5 + B * H * Dk * Dv * 40 / 2e12) * (2.2 if case["train"] else 1) > 15:
        return None
    f = lambda x: x.double()  # noqa: E731
    q, k, v = f(s["q"]) / math.sqrt(Dk), f(s["k"]).repeat_interleave(r, 2), f(s["v"]).repeat_interleave(r, 2)
    a = torch.exp(f(s["log_decay"]))[None, :, None, None]
    ends = (s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device="cuda")).long()
    on = (torch.arange(L, device="cuda")[:, None] < ends).double()[:, :, None, None, None]
    S = f(s["initial_state"]).clone() if case["start"] else torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device="cuda")
    T = torch.zeros_like(S)
    o = torch.zeros(B, L, H, Dv, dtype=torch.float64, device="cuda")
    do = f(s["do"]) if case["train"] else None
    dq = torch.zeros_like(q)
    dg = torch.zeros(H, dtype=torch.float64, device="cuda")
    ragged = case["ragged"]
    for t in range(L):
        if case["learn"]:
            T = torch.lerp(T, a * (T + S), on[t])
        new = torch.einsum("bhk,bhv->bhkv", k[:, t], v[:, t]).add_(S * a)
        S = torch.lerp(S, new, on[t]) if ragged else new
        o[:, t] = torch.matmul(q[:, t, :, None], S)[:, :, 0]
        if case["train"]:
            dq[:, t] = torch.matmul(S, do[:, t, :, :, None])[..., 0]
        if case["learn"]:
            live = on[t][:, :, 0, 0] if ragged else 1.0
            dg += ((torch.matmul(q[:, t, :, None], T)[:, :, 0] * do[:, t]).sum(-1) * live).sum(0)
    live = on[:, :, 0, 0, 0].t()[:, :, None, None]
    out = [o * live, S]
    if not case["train"]:
        return out
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    G = torch.zeros_like(S)
    for t in reversed(range(L)):
        new = torch.einsum("bhk,bhv->bhkv", q[:, t], do[:, t]).add_(G * a)
        # past a sequence's end nothing reaches its state
        G = new * on[t] if ragged else new
        dk[:, t] = torch.matmul(G, v[:, t, :, :, None])[..., 0]
        dv[:, t] = torch.matmul(k[:, t, :, None], G)[:, :, 0]
    shared = lambda x: (x * live).view(B, L, Hk, r, -1).sum(3)  # noqa: E731
    out += [dq * live / math.sqrt(Dk), shared(dk), shared(dv)]
    if case["start"]:
        out.append(G * a)
    if case["learn"]:
        out.append(dg)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "step":
        H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
        r = H // case["Hk"]
        a = torch.exp(s["log_decay"].double())
        head = torch.arange(H, device="cuda") // r
        k, v, q = s["k"].double()[:, head], s["v"].double()[:, head], s["q"].double() / math.sqrt(Dk)
        rows = s["slots"].tolist() if s["slots"] is not None else list(range(case["B"]))
        new, o = s["state"].double(), torch.zeros(case["B"], H, Dv, dtype=torch.float64, device="cuda")
        for b, n in enumerate(rows):
            if n >= 0:
                new[n] = a[:, None, None] * new[n] + torch.einsum("hk,hv->hkv", k[b], v[b])
                o[b] = torch.einsum("hk,hkv->hv", q[b], new[n])
        return [o, new]
    if case["op"] == "rotary":
        rot, L = case["rot"], case["L"]
        freq, amp = _frequencies(case)
        p = s["positions"].double() if s["positions"] is not None else torch.arange(L, dtype=torch.float64, device="cuda")[None]
        z = torch.polar(torch.full((1, 1), amp, dtype=torch.float64, device="cuda"), p[..., None] * freq)[:, :, None]

        def turn(x, by):
            x = x.double().clone()
            if case["interleaved"]:
                pair = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * by
                x[..., :rot] = torch.view_as_real(pair).flatten(-2)
            else:
                pair = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * by
                x[..., :rot // 2], x[..., rot // 2:rot] = pair.real, pair.imag
            return x

        out = [turn(s["q"], z), turn(s["k"], z)]
        return out + [turn(s["dq"], z.conj()), turn(s["dk"], z.conj())] if case["train"] else out
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = torch.sqrt(var + 1e-5)
    h = (x - mean) / sd
    w = s["weight"].double() if case["affine"] else torch.ones(case["C"], dtype=torch.float64, device="cuda")
    out = [h * w + (s["bias"].double() if case["affine"] else 0.0)]
    if case["train"]:
        dy = s["dy"].double()
        g = dy * w
        out.append((g - (g.sum(-1, keepdim=True) + h * (g * h).sum(-1, keepdim=True)) / case["C"]) / sd)
        if case["affine"]:
            out += [torch.einsum("rc,rc->c", dy, h), torch.einsum("rc->c", dy)]
    return out
