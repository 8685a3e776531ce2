"""Measured calls of the gated recurrent mixer's operators and of what serving a recurrent mixer needs beside them:

* ``scan`` — a gated linear recurrence over whole sequences (``gated_scan``), forward for prompts,
  forward and backward for training;
* ``step`` — its form for one token of every running request (``gated_scan_step``);
* ``qk`` — the norm of every head of queries and keys with rotary positions in the same pass
  (``qk_norm_rotary``), forward for serving, forward and backward with the weights' gradients for
  training;
* ``copy`` — slots of pools of states copied to others, all at once: requests forked, or the slots
  reordered in place (``copy_slots``);
* ``compact`` — running requests moved into the lowest slots (``compact_slots``).

The sizes are those of the mixers this package benchmarks (a 14 x 14 grid of 768 channels, a
128 x 128 grid of 256 channels, long sequences of up to 4096 channels), taken as sequences with
heads of 64 or 128 channels, and odd ones between them. ``run`` calls the package where ``own`` is
true; elsewhere it computes the same outputs from elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one sequence being answered, the 768-channel mixer: nothing but latency
        dict(name="step_one", op="step", dtype="bf16", B=1, C=768, pool=0, form="logit", complement=True, out_gate=True),
        # a serving step of 500 requests in a pool of 600 slots at 4096 channels, some slots idle
        dict(name="step_pool", op="step", dtype="bf16", B=500, C=4096, pool=600, form="logit", complement=True,
             out_gate=True),
        # prompts of unequal length in one batch that go on from earlier states
        dict(name="prompt_ragged", op="scan", dtype="bf16", B=16, L=1023, C=768, form="logit", complement=True,
             out_gate=True, ragged=True, start=True, train=False),
        # one long prompt at 4096 channels
        dict(name="prompt_long", op="scan", dtype="bf16", B=1, L=65536, C=4096, form="logit", complement=True,
             out_gate=True, ragged=False, start=False, train=False),
        # training on the 128 x 128 grid of 256 channels as a sequence
        dict(name="train_grid", op="scan", dtype="bf16", B=8, L=16384, C=256, form="logit", complement=True,
             out_gate=True, ragged=False, start=False, train=True),
        # a small 32-bit run with decays given as logarithms, an initial state, odd lengths and channels
        dict(name="train_f32_odd", op="scan", dtype="f32", B=2, L=1001, C=771, form="log", complement=False,
             out_gate=False, ragged=True, start=True, train=True),
        # the queries and keys of one token of 32 requests at unequal positions
        dict(name="qk_token", op="qk", dtype="bf16", B=32, L=1, H=12, Hk=4, D=64, rot=64, interleaved=False,
             positions="each", weights=True, train=False),
        # training on a long sequence of 4096 channels
        dict(name="qk_train", op="qk", dtype="bf16", B=1, L=65536, H=32, Hk=32, D=128, rot=128, interleaved=False,
             positions="none", weights=True, train=True),
        # neighbouring pairs, 50 of 80 features turned, odd lengths, half precision
        dict(name="qk_part", op="qk", dtype="f16", B=3, L=1021, H=5, Hk=5, D=80, rot=50, interleaved=True,
             positions="each", weights=True, train=True),
        # 8 prompts forked into 8 slots each: a layer's states of 12 heads of 64, and the positions
        dict(name="copy_fork", op="copy", N=224, row=49152, moves=64, how="fork"),
        # every slot reordered in place: states of 4096 channels, and the positions
        dict(name="copy_reorder", op="copy", N=2000, row=4096, moves=2000, how="permute"),
        # half of 224 requests have ended: states of 32 heads of 128
        dict(name="compact", op="compact", N=224, row=524288, live=0.5),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "step", "qk", "qk", "copy", "compact"])
    if op in ("copy", "compact"):
        row = _log_int(rng, 64, 524288)
        N = _log_int(rng, 2, min(2000, max(2, (1 << 26) // row)))
        if op == "compact":
            return dict(op=op, N=N, row=row, live=rng.uniform(0.1, 0.9))
        how = rng.choice(["fork", "permute", "clear"])
        return dict(op=op, N=N, row=row, moves=N if how == "permute" else rng.randrange(1, max(1, N // 2) + 1), how=how)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "qk":
        B, Hk = _log_int(rng, 1, 32), rng.choice([1, 2, 4, 6, 8])
        H = Hk * rng.choice([1, 1, 2, 3])
        D = rng.choice([64, 128, 80, rng.randrange(16, 257)])
        rot = max(2, min(D, rng.choice([D, D // 2, rng.randrange(2, D + 1)])) // 2 * 2)
        L = _log_int(rng, 1, max(1, min(65536, (1 << 26) // (B * H * D))))
        return dict(op=op, dtype=dtype, B=B, L=L, H=H, Hk=Hk, D=D, rot=rot, interleaved=rng.random() < 0.5,
                    positions=rng.choice(["none", "each"]), weights=rng.random() < 0.8, train=rng.random() < 0.5)
    form = rng.choice(["logit", "logit", "log"])
    kind = dict(form=form, complement=rng.random() < 0.5, out_gate=rng.random() < 0.5)
    C = rng.choice([256, 768, 1024, _log_int(rng, 16, 4096)])
    if op == "step":
        B = _log_int(rng, 1, 512)
        return dict(op=op, dtype=dtype, B=B, C=C, pool=rng.choice([0, B + 3]), **kind)
    B = _log_int(rng, 1, 32)
    L = _log_int(rng, 1, max(1, min(65536, (1 << 26) // (B * C))))
    return dict(op=op, dtype=dtype, B=B, L=L, C=C, **kind, ragged=rng.random() < 0.4, start=rng.random() < 0.4,
                train=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs


def _randn(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _gate(gen, shape, form, dtype):
    """Memories of 16 tokens to 4096 spread over the channels, moved by each token."""
    memory = 2.0 ** torch.linspace(4.0, 12.0, shape[-1], device="cuda")
    if form == "logit":
        return (torch.log(memory - 1) + 1.5 * _randn(gen, shape)).to(dtype)
    return (-torch.exp(0.5 * _randn(gen, shape)) / memory).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, op = {"case": case}, case["op"]
    if op in ("copy", "compact"):
        N = case["N"]
        s["pools"] = [_randn(gen, (N, case["row"])), torch.randint(0, 100000, (N,), generator=gen, device="cuda")]
        order = torch.randperm(N, generator=gen, device="cuda").to(torch.int32)
        if op == "compact":
            alive = max(1, int(round(case["live"] * N)))
            s["live"] = order < alive
        elif case["how"] == "permute":
            s["source"], s["target"] = order, torch.arange(N, dtype=torch.int32, device="cuda")
        else:
            n = case["moves"]
            s["target"] = order[:n].contiguous()
            if case["how"] == "clear":
                s["source"] = torch.full_like(s["target"], -1)
            else:  # up to eight copies of each prompt, into slots that are no prompt's
                prompts = order[n:]
                which = torch.arange(n, device="cuda") // 8 % max(1, prompts.numel())
                s["source"] = prompts[which].contiguous()
        return s
    dt = DTYPES[case["dtype"]]
    if op == "qk":
        B, L, H, Hk, D = (case[n] for n in ("B", "L", "H", "Hk", "D"))
        s["q"], s["k"] = (2 * _randn(gen, (B, L, H, D))).to(dt), (2 * _randn(gen, (B, L, Hk, D))).to(dt)
        s["q_weight"] = (1 + 0.2 * _randn(gen, (D,))).to(dt) if case["weights"] else None
        s["k_weight"] = (1 + 0.2 * _randn(gen, (D,))).to(dt) if case["weights"] else None
        s["positions"] = None
        if case["positions"] == "each":  # each request goes on from where its cache ends
            s["positions"] = (torch.randint(0, 100000, (B, 1), generator=gen, device="cuda")
                              + torch.arange(L, device="cuda"))
        if case["train"]:
            s["dq"], s["dk"] = _randn(gen, (B, L, H, D), dt), _randn(gen, (B, L, Hk, D), dt)
        # turns per position in units of 2^-64, so that whole turns drop out exactly
        freq = [10000.0 ** (-2.0 * i / case["rot"]) for i in range(case["rot"] // 2)]
        s["turns"] = torch.tensor([int(f / (2 * math.pi) * 2.0 ** 64) for f in freq], device="cuda")
        return s
    B, C = case["B"], case["C"]
    shape = (B, C) if op == "step" else (B, case["L"], C)
    s["x"], s["gate"] = _randn(gen, shape, dt), _gate(gen, shape, case["form"], dt)
    s["out_gate"] = _randn(gen, shape, dt) if case["out_gate"] else None
    if op == "step":
        N = case["pool"] or B
        s["state"] = _randn(gen, (N, C))
        s["new_state"] = s["state"].clone()
        s["slots"] = None
        if case["pool"]:  # every seventh request has no slot and is passed over
            s["slots"] = torch.randperm(N, generator=gen, device="cuda")[:B].to(torch.int32)
            s["slots"][5::7] = -1
        return s
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, case["L"] + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        s["lengths"][0] = case["L"]
        s["lengths"][1:2] = 0
        s["lengths"][2:3] = 1
    s["initial_state"] = _randn(gen, (B, C)) if case["start"] else None
    if case["train"]:
        s["dy"] = _randn(gen, shape, dt)
    return s


# ---------------------------------------------------------------- the plain forms, 32 bits


def _decays(gate, form):
    """(a, 1 - a), each without cancellation."""
    g = gate.float()
    return (torch.sigmoid(g), torch.sigmoid(-g)) if form == "logit" else (torch.exp(g), -torch.expm1(g))


def _chain(u, b):
    """h_t = (1 - u_t) h_{t-1} + b_t along axis 1 from zero, by doubling: after a pass each token has gathered twice as many.
    Decays go as what they take away, which keeps its digits where a decay near 1 would lose them token by token."""
    d = 1
    while d < u.shape[1]:
        b = torch.cat((b[:, :d], b[:, d:] + (b[:, :-d] - u[:, d:] * b[:, :-d])), 1)
        u = torch.cat((u[:, :d], u[:, d:] + (u[:, :-d] - u[:, d:] * u[:, :-d])), 1)
        d *= 2
    return b


def _plain_scan(s):
    case, x = s["case"], s["x"]
    B, L, C = x.shape
    a, u = _decays(s["gate"], case["form"])
    xf = x.float()
    live = None
    if case["ragged"]:
        live = (torch.arange(L, device=x.device) < s["lengths"][:, None])[..., None]
        a, u, xf = torch.where(live, a, 1.0), torch.where(live, u, 0.0), torch.where(live, xf, 0.0)
    h0 = s["initial_state"] if case["start"] else torch.zeros(B, C, device=x.device)
    b = u * xf if case["complement"] else xf
    b = torch.cat(((b[:, 0] + (h0 - u[:, 0] * h0))[:, None], b[:, 1:]), 1)
    h = _chain(u, b)
    y, o = h, None
    if case["out_gate"]:
        o = s["out_gate"].float()
        y = h * (o * torch.sigmoid(o))
    keep = (lambda t: t.to(x.dtype)) if live is None else (lambda t: torch.where(live, t, 0.0).to(x.dtype))
    out = [keep(y), h[:, -1].clone()]
    if not case["train"]:
        return out
    dy = s["dy"].float()
    dh = dy if live is None else torch.where(live, dy, 0.0)
    if o is not None:
        sig = torch.sigmoid(o)
        do = keep(dh * h * (sig * (1 + o * (1 - sig))))
        dh = dh * (o * sig)
    after = torch.cat((u[:, 1:], torch.zeros_like(u[:, :1])), 1)
    G = _chain(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    dx = G * u if case["complement"] else G
    da = G * (before - xf) if case["complement"] else G * before
    dg = da * a * u if case["form"] == "logit" else da * a
    out += [keep(dx), keep(dg)]
    if o is not None:
        out.append(do)
    if case["start"]:
        out.append(a[:, 0] * G[:, 0])
    return out


def _plain_step(s):
    case, slots, state = s["case"], s["slots"], s["state"]
    at = slots.long().clamp(min=0) if slots is not None else torch.arange(s["x"].shape[0], device=state.device)
    a, u = _decays(s["gate"], case["form"])
    x = s["x"].float()
    h = a * state[at] + (u * x if case["complement"] else x)
    y = h
    if case["out_gate"]:
        o = s["out_gate"].float()
        y = h * (o * torch.sigmoid(o))
    if slots is None:
        s["new_state"].copy_(h)
        return [y.to(s["x"].dtype), s["new_state"]]
    on = slots >= 0
    s["new_state"][at[on]] = h[on]
    return [torch.where(on[:, None], y, 0.0).to(s["x"].dtype), s["new_state"]]


def _plain_turn(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_qk(s):
    case, q = s["case"], s["q"]
    p = s["positions"] if s["positions"] is not None else torch.arange(q.shape[1], device=q.device)[None]
    part = (p[..., None] * s["turns"]) >> 32  # 64-bit products wrap: what is left is the turn's fraction
    angle = part.float() * (2 * math.pi / 2.0 ** 32)
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
    rot, inter = case["rot"], case["interleaved"]

    def normed(x, w):
        r = torch.rsqrt((x.float() ** 2).mean(-1, keepdim=True) + EPS)
        h = x.float() * r
        n = h if w is None else h * w.float()
        return h, r, _plain_turn(n, cos, sin, rot, inter).to(x.dtype)

    def back(dy, x, w, h, r):
        t = _plain_turn(dy.float(), cos, -sin, rot, inter)  # a turn's transpose is the turn back
        g = t if w is None else t * w.float()
        dx = r * (g - h * (g * h).mean(-1, keepdim=True))
        return dx.to(x.dtype), None if w is None else (t * h).sum((0, 1, 2)).to(w.dtype)

    hq, rq, yq = normed(s["q"], s["q_weight"])
    hk, rk, yk = normed(s["k"], s["k_weight"])
    out = [yq, yk]
    if case["train"]:
        dq, dwq = back(s["dq"], s["q"], s["q_weight"], hq, rq)
        dk, dwk = back(s["dk"], s["k"], s["k_weight"], hk, rk)
        out += [dq, dk] + ([dwq, dwk] if case["weights"] else [])
    return out


def _plain_copy(s):
    source, target = s["source"].long(), s["target"].long()
    for pool in s["pools"]:
        if s["case"]["how"] == "clear":
            pool.index_fill_(0, target, 0)
        else:
            pool.index_copy_(0, target, pool[source])
    return list(s["pools"])


def _plain_compact(s):
    live = s["live"]
    slot = torch.arange(live.numel(), device=live.device)
    low = slot < live.sum()
    holes, movers = (~live & low).nonzero()[:, 0], (live & ~low).nonzero()[:, 0]
    new = torch.where(live, slot, -1)
    new[movers] = holes
    for pool in s["pools"]:
        pool.index_copy_(0, holes, pool[movers])
    return [*s["pools"], new.to(torch.int32)]


# ---------------------------------------------------------------- one pass


def _own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "copy":
        from nvsubquadratic_b200.state_pool import copy_slots

        copy_slots(s["pools"], s["source"], s["target"])
        return list(s["pools"])
    if op == "compact":
        from nvsubquadratic_b200.state_pool import compact_slots

        new = compact_slots(s["pools"], s["live"])
        return [*s["pools"], new]
    if op == "qk":
        from nvsubquadratic_b200.qk_norm import qk_norm_rotary

        args = [s["q"], s["k"], s["q_weight"], s["k_weight"]]
        if case["train"]:
            args = [a.detach().requires_grad_() if a is not None else None for a in args]
        out = qk_norm_rotary(*args, s["turns"], eps=EPS, positions=s["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return list(out)
        return [*out, *torch.autograd.grad(out, [a for a in args if a is not None], [s["dq"], s["dk"]])]
    kind = dict(form=case["form"], complement=case["complement"])
    if op == "step":
        from nvsubquadratic_b200.gated_scan import gated_scan_step

        y = gated_scan_step(s["x"], s["gate"], s["state"], out_gate=s["out_gate"], slots=s["slots"],
                            out_state=s["new_state"], **kind)
        return [y, s["new_state"]]
    from nvsubquadratic_b200.gated_scan import gated_scan

    names = ["x", "gate", "out_gate", "initial_state"]
    given = {n: s[n] for n in names}
    if case["train"]:
        given = {n: t.detach().requires_grad_() if t is not None else None for n, t in given.items()}
    y, state = gated_scan(given["x"], given["gate"], out_gate=given["out_gate"], lengths=s["lengths"],
                          initial_state=given["initial_state"], return_state=True, **kind)
    if not case["train"]:
        return [y, state]
    return [y, state, *torch.autograd.grad(y, [t for t in given.values() if t is not None], s["dy"])]


def run(state):
    if own:
        return _own(state)
    forms = {"scan": _plain_scan, "step": _plain_step, "qk": _plain_qk, "copy": _plain_copy, "compact": _plain_compact}
    return forms[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op in ("copy", "compact"):
        row, N = 4 * case["row"] + 8, case["N"]
        if op == "compact":  # dead slots lie anywhere: of the lowest `alive` slots that share is free
            alive = max(1, int(round(case["live"] * N)))
            return {"bytes": 2 * row * max(1, alive * (N - alive) // N) + 5 * N, "flops": 0}
        n = case["moves"]
        read = {"permute": n, "fork": max(1, min(-(-n // 8), N - n)), "clear": 0}[case["how"]]
        return {"bytes": row * (n + read) + 8 * n, "flops": 0}
    e = 4 if case["dtype"] == "f32" else 2
    if op == "qk":
        n = case["B"] * case["L"] * (case["H"] + case["Hk"]) * case["D"]
        places = 8 * case["B"] * case["L"] if case["positions"] == "each" else 0
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * e * n * passes + places, "flops": 7 * n + (12 * n if case["train"] else 0)}
    B, C, gates = case["B"], case["C"], 1 if case["out_gate"] else 0
    if op == "step":
        on = B - (len(range(5, B, 7)) if case["pool"] else 0)
        return {"bytes": C * (8 * on + e * (on * (2 + gates) + B)) + (4 * B if case["pool"] else 0), "flops": 12 * on * C}
    # ragged lengths are uniform over 0..L: the first is L, the second 0, the third 1
    L = case["L"]
    tokens = B * L
    if case["ragged"]:
        tokens = L + (1 if B > 2 else 0) + max(0, B - 3) * L // 2
    states = 4 * B * C
    byts = e * C * (tokens * (2 + gates) + B * L) + states * (2 if case["start"] else 1)
    flops = 14 * tokens * C
    if case["train"]:
        byts += e * C * (tokens + B * L * (2 + gates)) + (states if case["start"] else 0)
        flops += 24 * tokens * C
    return {"bytes": byts, "flops": flops}


# ---------------------------------------------------------------- 64 bits, from the definitions


def _exact_scan(case, s):
    """The recurrence token by token, and its derivative token by token backwards."""
    B, L, C = case["B"], case["L"], case["C"]
    if L * (1.2e-4 + B * C * 1e-10) * (2.5 if case["train"] else 1) > 18 or 8 * B * L * C > 4e9:
        return None
    g, x = s["gate"].double(), s["x"].double()
    a = 1 / (1 + torch.exp(-g)) if case["form"] == "logit" else torch.exp(g)
    ends = (s["lengths"] if case["ragged"] else torch.full((B,), L, device="cuda")).long()
    o = s["out_gate"].double() if case["out_gate"] else None
    act = o / (1 + torch.exp(-o)) if o is not None else None
    h = s["initial_state"].double() if case["start"] else torch.zeros(B, C, dtype=torch.float64, device="cuda")
    seen = torch.empty(L + 1, B, C, dtype=torch.float64, device="cuda")
    seen[0] = h
    for t in range(L):
        new = a[:, t] * h + (1 - a[:, t]) * x[:, t] if case["complement"] else a[:, t] * h + x[:, t]
        h = torch.where((t < ends)[:, None], new, h) if case["ragged"] else new
        seen[t + 1] = h
    on = (torch.arange(L, device="cuda") < ends[:, None])[..., None]
    hs = seen[1:].transpose(0, 1)
    y = torch.where(on, hs * act if act is not None else hs, 0.0)
    out = [y, h]
    if not case["train"]:
        return out
    dy = torch.where(on, s["dy"].double(), 0.0)
    dh = dy * act if act is not None else dy
    dx, dg = torch.zeros_like(x), torch.zeros_like(x)
    c = torch.zeros(B, C, dtype=torch.float64, device="cuda")
    for t in range(L - 1, -1, -1):
        G = dh[:, t] + c
        at = a[:, t]
        if case["complement"]:
            dx[:, t] = (1 - at) * G
            da = G * (seen[t] - x[:, t])
        else:
            dx[:, t] = G
            da = G * seen[t]
        dg[:, t] = da * at * (1 - at) if case["form"] == "logit" else da * at
        c = torch.where((t < ends)[:, None], at * G, c) if case["ragged"] else at * G
    out += [torch.where(on, dx, 0.0), torch.where(on, dg, 0.0)]
    if o is not None:
        sig = 1 / (1 + torch.exp(-o))
        out.append(torch.where(on, dy * hs * (sig + o * sig * (1 - sig)), 0.0))
    if case["start"]:
        out.append(c)
    return out


def _exact_qk(case, s):
    """Rows divided by their root mean square, and pairs turned as products of complex numbers."""
    if case["B"] * case["L"] * case["H"] * case["D"] > 3e8:
        return None
    rot = case["rot"]
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    p = s["positions"] if s["positions"] is not None else torch.arange(case["L"], device="cuda")[None]
    unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), p.double()[..., None] * freq)[:, :, None]
    i = torch.arange(rot // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)

    def turn(x, z):
        y = x.clone()
        w = torch.complex(x[..., first], x[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    out, back, weights = [], [], []
    for n in ("q", "k"):
        x = s[n].double()
        w = s[n + "_weight"].double() if case["weights"] else torch.ones(case["D"], dtype=torch.float64, device="cuda")
        rms = (x.square().sum(-1, keepdim=True) / case["D"] + EPS).sqrt()
        out.append(turn(x / rms * w, unit))
        if case["train"]:
            t = turn(s["d" + n].double(), unit.conj())
            g = t * w
            back.append(g / rms - x * (g * x).sum(-1, keepdim=True) / (case["D"] * rms ** 3))
            weights.append((t * x / rms).sum((0, 1, 2)))
    return out + back + (weights if case["weights"] else [])


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "scan":
        return _exact_scan(case, s)
    if op == "qk":
        return _exact_qk(case, s)
    if op == "step":
        g, x = s["gate"].double(), s["x"].double()
        a = 1 / (1 + torch.exp(-g)) if case["form"] == "logit" else torch.exp(g)
        y, new = torch.zeros_like(x), s["state"].double()
        for b in range(case["B"]):
            at = b if s["slots"] is None else int(s["slots"][b])
            if at >= 0:
                new[at] = a[b] * new[at] + ((1 - a[b]) * x[b] if case["complement"] else x[b])
                y[b] = new[at]
        if case["out_gate"]:
            o = s["out_gate"].double()
            y = y * o / (1 + torch.exp(-o))
        return [y, new]
    # copies of numbers: what every slot holds afterwards, slot by slot
    N = case["N"]
    held, new = list(range(N)), None
    if op == "copy":
        for a, b in zip(s["source"].tolist(), s["target"].tolist()):
            held[b] = a
    else:
        live = s["live"].tolist()
        high = [i for i in range(sum(live), N) if live[i]]
        new = [i if live[i] else -1 for i in range(N)]
        for i in range(sum(live)):
            if not live[i]:
                held[i] = high.pop(0)
                new[held[i]] = i
    at = torch.tensor(held, device="cuda")
    state = torch.where((at >= 0)[:, None], s["pools"][0][at.clamp(min=0)], 0.0)
    position = torch.where(at >= 0, s["pools"][1][at.clamp(min=0)], 0)
    return [state, position] + ([torch.tensor(new, dtype=torch.int32)] if new is not None else [])
