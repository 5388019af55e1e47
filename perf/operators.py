"""Workloads of the gated linear recurrence, its single-token step and the group norm with an activation.

``listed()`` names the fixed cases, ``draw(rng)`` gives further ones of the same ranges.  ``prepare`` makes what a
program has in hand before the call, ``run`` is one pass: with ``own`` through the framework's operators, without it in
elementary torch operations.  A training pass is a forward and a backward and returns the gradients too.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 64e-5                     # what the RWKV output stages use


def listed():
    return [
        # a short prompt of one user through a 0.1B model: launches and latency
        {"name": "rec-prompt-short", "op": "recurrence", "train": False, "dtype": "bf16", "gate": "sigmoid", "B": 1, "T": 37, "C": 768,
         "starts": 0.0, "ragged": False, "halves": False},
        # one prompt of 2000 tokens at the width of a 2.9B model
        {"name": "rec-prompt-2000", "op": "recurrence", "train": False, "dtype": "bf16", "gate": "decay", "B": 1, "T": 2000, "C": 2560,
         "starts": 0.0, "ragged": False, "halves": False},
        # one very long document: few channels in parallel, a long axis
        {"name": "rec-document", "op": "recurrence", "train": False, "dtype": "bf16", "gate": "sigmoid", "B": 1, "T": 32768, "C": 2048,
         "starts": 0.0, "ragged": False, "halves": False},
        # a training step of one layer of a 1.5B model on packed documents (the benchmark's batch and length)
        {"name": "rec-train-1.5B", "op": "recurrence", "train": True, "dtype": "bf16", "gate": "sigmoid", "B": 8, "T": 4096, "C": 2048,
         "starts": 1 / 512, "ragged": True, "halves": False},
        # training where one projection makes both operands, which are then halves of its rows
        {"name": "rec-train-halves", "op": "recurrence", "train": True, "dtype": "bf16", "gate": "decay", "B": 4, "T": 1024, "C": 2048,
         "starts": 0.0, "ragged": False, "halves": True},
        # fp32 training with odd sizes: a gradient check, a small experiment
        {"name": "rec-train-fp32-odd", "op": "recurrence", "train": True, "dtype": "fp32", "gate": "decay", "B": 3, "T": 1023, "C": 1001,
         "starts": 1 / 256, "ragged": True, "halves": False},
        # one token of one user: launches and latency
        {"name": "step-1", "op": "step", "dtype": "bf16", "gate": "sigmoid", "B": 1, "C": 2048, "starts": 0.0, "ragged": False},
        # one token of many users, some of them starting anew, some without a token
        {"name": "step-1024", "op": "step", "dtype": "fp32", "gate": "decay", "B": 1024, "C": 2560, "starts": 1 / 64, "ragged": True},
        # the output stage of one decoded token
        {"name": "norm-token", "op": "norm", "train": False, "dtype": "bf16", "rows": 1, "C": 2048, "groups": 32, "gated": True,
         "activation": "silu", "part": False},
        # the output stage of a training step (heads of 64 channels, gated by silu as in RWKV-5.2 and 6)
        {"name": "norm-train-1.5B", "op": "norm", "train": True, "dtype": "bf16", "rows": 32768, "C": 2048, "groups": 32, "gated": True,
         "activation": "silu", "part": False},
        # fp32 training with odd sizes: groups of 60 channels
        {"name": "norm-train-fp32-odd", "op": "norm", "train": True, "dtype": "fp32", "rows": 1021, "C": 1020, "groups": 17, "gated": True,
         "activation": "sigmoid", "part": False},
        # wide groups without a gate, over a part of wider rows
        {"name": "norm-wide-groups", "op": "norm", "train": False, "dtype": "bf16", "rows": 8190, "C": 4096, "groups": 8, "gated": False,
         "activation": "silu", "part": True},
    ]


OPS = ("recurrence",) * 6 + ("step",) * 2 + ("norm",) * 4
MOST = 1 << 26                  # elements of a stream in 16 bits; half of it in 32


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(OPS)
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    most = MOST if dtype == "bf16" else MOST // 2
    case = {"op": op, "dtype": dtype}
    if op == "norm":
        train = rng.random() < 0.5
        size = rng.choice((_log(rng, 16, 512), 64, 8 * _log(rng, 2, 64)))
        groups = max(1, min(_log(rng, 1, 64), 8192 // size))
        rows = min(_log(rng, 1, 32768), most // (size * groups))
        case.update(train=train, rows=rows, C=size * groups, groups=groups, gated=rng.random() < 0.7,
                    activation=rng.choice(("none", "sigmoid", "silu")), part=rng.random() < 0.3)
        return case
    C = 64 * _log(rng, 4, 80) if rng.random() < 0.6 else _log(rng, 250, 4100)
    gate = rng.choice(("sigmoid", "decay"))
    if op == "step":
        case.update(gate=gate, B=_log(rng, 1, 1024), C=C, starts=rng.choice((0.0, 1 / 64)), ragged=rng.random() < 0.3)
        return case
    train = rng.random() < 0.5
    T = _log(rng, 1, 8192 if train else 32768)
    B = max(1, min(_log(rng, 1, 16), most // (T * C)))
    T = min(T, most // (B * C))
    case.update(train=train, gate=gate, B=B, T=T, C=C, starts=rng.choice((0.0, 0.0, 1 / 512, 1 / 64)), ragged=rng.random() < 0.4,
                halves=rng.random() < 0.3)
    return case


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n, streams = case["rows"] * case["C"], 2 + case["gated"]
        if not case["train"]:
            return {"bytes": n * streams * e + 2 * case["C"] * e, "flops": n * (10 + 5 * case["gated"])}
        return {"bytes": n * 2 * streams * e + 4 * case["C"] * e, "flops": n * (28 + 12 * case["gated"])}
    rows = case["B"]
    states = rows * case["C"] * 4
    if case["op"] == "step":
        return {"bytes": rows * case["C"] * 3 * e + 2 * states + (8 * rows if case["ragged"] or case["starts"] else 0),
                "flops": rows * case["C"] * 10}
    n = rows * case["T"] * case["C"]
    flags = rows * (case["T"] + 4)
    if not case["train"]:
        return {"bytes": n * 3 * e + 2 * states + flags, "flops": n * 10}
    return {"bytes": n * 6 * e + 4 * states + flags, "flops": n * 30}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _gate_values(g, case, *lead):
    """What a model feeds the gates: forget gates that mostly keep, or RWKV-6's log-log decays over the channels."""
    C = case["C"]
    if case["gate"] == "sigmoid":
        return 2.0 + 1.5 * _normal(g, *lead, C)
    return torch.linspace(-6.0, -1.0, C, device="cuda") + 0.5 * _normal(g, *lead, C)


def _flags(g, case, T):
    B = case["B"]
    starts = torch.rand((B, T), generator=g, device="cuda") < case["starts"]
    length = torch.full((B,), T, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        length = torch.randint(0, T + 1, (B,), generator=g, device="cuda").to(torch.int32)
    return length, starts


def prepare(case, seed):
    g, dtype, C = _generator(seed), DTYPES[case["dtype"]], case["C"]
    if case["op"] == "norm":
        rows = case["rows"]
        x = 0.5 * torch.linspace(-1.0, 1.0, C, device="cuda") + _normal(g, rows, C)
        gate = _normal(g, rows, C) if case["gated"] else None
        if case["part"]:                        # columns of wider rows, as a projection for several uses leaves them
            wide = torch.zeros(rows, 2 * C + 64, dtype=dtype, device="cuda")
            wide[:, :C] = x
            x = wide[:, :C]
            if gate is not None:
                wide[:, C:2 * C] = gate
                gate = wide[:, C:2 * C]
        else:
            x = x.to(dtype)
            gate = None if gate is None else gate.to(dtype)
        weight = (1.0 + 0.1 * _normal(g, C)).to(dtype)
        bias = (0.1 * _normal(g, C)).to(dtype)
        state = {"case": case, "x": x, "gate": gate, "weight": weight, "bias": bias}
        if case["train"]:
            state["gy"] = _normal(g, rows, C).to(dtype)
            for name in ("x", "gate", "weight", "bias"):
                if state[name] is not None:
                    state[name] = state[name].detach().requires_grad_(True)
        return state
    B = case["B"]
    s = _normal(g, B, C)
    if case["op"] == "step":
        length, starts = _flags(g, case, 1)
        x, f = _normal(g, B, C).to(dtype), _gate_values(g, case, B).to(dtype)
        if not (case["ragged"] or case["starts"]):
            length = starts = None
        return {"case": case, "x": x, "f": f, "s": s, "length": length, "starts": starts}
    T = case["T"]
    length, starts = _flags(g, case, T)
    if case["halves"]:
        both = torch.empty(B, T, 2 * C, dtype=dtype, device="cuda")
        x, f = both[..., :C], both[..., C:]
        x.copy_(_normal(g, B, T, C))
        f.copy_(_gate_values(g, case, B, T))
    else:
        x, f = _normal(g, B, T, C).to(dtype), _gate_values(g, case, B, T).to(dtype)
    state = {"case": case, "x": x, "f": f, "s": s, "length": length, "starts": starts}
    if case["train"]:
        state["gy"], state["gs"] = _normal(g, B, T, C).to(dtype), _normal(g, B, C)
        for name in ("x", "f", "s"):
            state[name] = state[name].detach().requires_grad_(True)
    return state


def run(state):
    case = state["case"]
    kind = "norm" if case["op"] == "norm" else case["op"]
    return (_OWN if own else _PLAIN)[kind](case, state)


# ---------------------------------------------------------------------------------- the framework's operators
def _own_recurrence(case, st):
    from jaxrwkv_b200.gated_recurrence import gated_recurrence
    s_out, out = gated_recurrence(st["x"], st["f"], st["s"], st["length"], st["starts"], gate=case["gate"])
    if not case["train"]:
        return [s_out, out]
    return [s_out, out, *torch.autograd.grad((s_out, out), (st["x"], st["f"], st["s"]), (st["gs"], st["gy"]))]


def _own_step(case, st):
    from jaxrwkv_b200.gated_recurrence import gated_recurrence_step
    return list(gated_recurrence_step(st["x"], st["f"], st["s"], st["starts"], st["length"], gate=case["gate"]))


def _own_norm(case, st):
    from jaxrwkv_b200.group_norm import group_norm_act
    out = group_norm_act(st["x"], st["weight"], st["bias"], case["groups"], gate=st["gate"], activation=case["activation"], eps=EPS)
    if not case["train"]:
        return [out]
    leaves = [st[n] for n in ("x", "gate", "weight", "bias") if st[n] is not None]
    return [out, *torch.autograd.grad(out, leaves, st["gy"])]


# ---------------------------------------------------------------------------------- plain forms
def _coefficients(case, x, f):
    """(a, u, weight of x in u) of h = a h + u, in 32 bits."""
    if case["gate"] == "sigmoid":
        a, w = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
        return a, w * x, w
    return torch.exp(-torch.exp(f)), x, None


def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1 from zero, by doubling."""
    n, T = 1, a.shape[1]
    while n < T:
        u = torch.cat([u[:, :n], u[:, n:] + a[:, n:] * u[:, :-n]], dim=1)
        if 2 * n < T:
            a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], dim=1)
        n *= 2
    return u


def _plain_recurrence(case, st):
    with torch.no_grad():
        B, T, C = st["x"].shape
        x, f, s = st["x"].float(), st["f"].float(), st["s"]
        length = st["length"].long()
        a, u, w = _coefficients(case, x, f)
        kept = torch.where(st["starts"][:, :, None], torch.zeros_like(a), a)      # what a token keeps of the state
        first = u.clone()
        first[:, 0] += kept[:, 0] * s
        h = _scan(kept, first)
        del first, u
        rows = torch.arange(B, device=x.device)
        last = (length - 1).clamp(min=0)
        s_out = torch.where((length > 0)[:, None], h[rows, last], s)
        if not case["train"]:
            return [s_out, h.to(st["x"].dtype)]
        g = st["gy"].to(torch.float32, copy=True)
        g[rows, last] += torch.where((length > 0)[:, None], st["gs"], torch.zeros_like(st["gs"]))
        behind = torch.cat([kept[:, 1:], torch.zeros_like(kept[:, :1])], dim=1)
        dh = _scan(behind.flip(1), g.flip(1)).flip(1)
        del behind, g
        hp = torch.cat([s[:, None], h[:, :-1]], dim=1)
        hp = torch.where(st["starts"][:, :, None], torch.zeros_like(hp), hp)
        ds = kept[:, 0] * dh[:, 0] + torch.where((length == 0)[:, None], st["gs"], torch.zeros_like(st["gs"]))
        if case["gate"] == "sigmoid":
            dx, df = w * dh, dh * (hp - x) * a * w
        else:
            dx, df = dh, -dh * hp * torch.exp(f) * a
        out_type = st["x"].dtype
        return [s_out, h.to(out_type), dx.to(out_type), df.to(out_type), ds]


def _plain_step(case, st):
    x, f, s = st["x"].float(), st["f"].float(), st["s"]
    a, u, _ = _coefficients(case, x, f)
    if st["starts"] is not None:
        a = torch.where(st["starts"].reshape(-1, 1), torch.zeros_like(a), a)
    h = a * s + u
    s_out = h if st["length"] is None else torch.where((st["length"] > 0)[:, None], h, s)
    return [s_out, h.to(st["x"].dtype)]


def _act(name, z):
    """(act(z), act'(z))."""
    if name == "none":
        return z, torch.ones_like(z)
    p = 1.0 / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return p, p * (1.0 - p)
    return z * p, p * (1.0 + z * (1.0 - p))


def _plain_norm(case, st):
    with torch.no_grad():
        dtype, rows, C, G = st["x"].dtype, case["rows"], case["C"], case["groups"]
        x = st["x"].float().reshape(rows, G, C // G)
        x = x - x.mean(dim=2, keepdim=True)
        rstd = 1.0 / torch.sqrt((x * x).mean(dim=2, keepdim=True) + EPS)
        xh = (x * rstd).reshape(rows, C)
        weight = st["weight"].float()
        n = xh * weight + st["bias"].float()
        if case["gated"]:
            p, dp = _act(case["activation"], st["gate"].float())
            out = n * p
        else:
            out, dn = _act(case["activation"], n)
        if not case["train"]:
            return [out.to(dtype)]
        gy = st["gy"].float()
        grads = []
        if case["gated"]:
            dn = gy * p
            grads.append((gy * n * dp).to(dtype))
        else:
            dn = gy * dn
        dw, db = (dn * xh).sum(0, dtype=torch.float64), dn.sum(0, dtype=torch.float64)
        dxh, xh = (dn * weight).reshape(rows, G, C // G), xh.reshape(rows, G, C // G)
        dx = rstd * (dxh - dxh.mean(dim=2, keepdim=True) - xh * (dxh * xh).mean(dim=2, keepdim=True))
        return [out.to(dtype), dx.reshape(rows, C).to(dtype), *grads, dw.to(dtype), db.to(dtype)]


_OWN = {"recurrence": _own_recurrence, "step": _own_step, "norm": _own_norm}
_PLAIN = {"recurrence": _plain_recurrence, "step": _plain_step, "norm": _plain_norm}


# ---------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, st) if case["op"] == "norm" else _exact_recurrence(case, st)


def _exact_recurrence(case, st):
    """Token by token, the gradients by walking back with what a token's state is worth."""
    step = case["op"] == "step"
    B, C = case["B"], case["C"]
    T = 1 if step else case["T"]
    x, f = st["x"].double().reshape(B, T, C), st["f"].double().reshape(B, T, C)
    s, dev = st["s"].double(), st["x"].device
    length = torch.full((B,), T, device=dev) if st["length"] is None else st["length"].long()
    starts = torch.zeros(B, T, dtype=torch.bool, device=dev) if st["starts"] is None else st["starts"]
    goes_on = (~starts).double()[:, :, None]
    sigmoid = case["gate"] == "sigmoid"
    keep = torch.sigmoid(f) if sigmoid else torch.exp(-torch.exp(f))
    enter = torch.sigmoid(-f) if sigmoid else None
    ends = (length[:, None] - 1 == torch.arange(T, device=dev)).double()[:, :, None]
    hs = torch.empty_like(x)
    h, s_out = s, s * (length == 0).double()[:, None]
    linear = keep * goes_on
    add = enter * x if sigmoid else x
    for t in range(T):
        h = torch.addcmul(add[:, t], linear[:, t], h, out=hs[:, t])
    s_out = s_out + (hs * ends).sum(1)
    if step:
        return [s_out, hs[:, 0]]
    if not case["train"]:
        return [s_out, hs]
    worth = st["gy"].double() + ends * st["gs"].double()[:, None]
    for t in range(T - 2, -1, -1):
        worth[:, t].addcmul_(linear[:, t + 1], worth[:, t + 1])
    before = torch.cat([s[:, None], hs[:, :-1]], 1) * goes_on
    ds = linear[:, 0] * worth[:, 0] + st["gs"].double() * (length == 0).double()[:, None]
    if sigmoid:
        return [s_out, hs, worth * enter, worth * (before - x) * keep * enter, ds]
    return [s_out, hs, worth, -(worth * before) * torch.exp(f - torch.exp(f)), ds]


def _exact_norm(case, st):
    """The definition in 64 bits, its gradients by autograd, some rows at a time (a row depends on no other)."""
    C, G = case["C"], case["groups"]
    act = {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}[case["activation"]]
    weight, bias = (st[n].detach().double().requires_grad_(True) for n in ("weight", "bias"))
    outs, gxs, ggs, sums = [], [], [], [torch.zeros_like(weight), torch.zeros_like(bias)]
    for lo in range(0, case["rows"], 8192):
        cut = slice(lo, lo + 8192)
        x = st["x"].detach()[cut].double().requires_grad_(True)
        leaves = [x, weight, bias]
        with torch.enable_grad():
            z = x.unflatten(1, (G, C // G))
            var, mean = torch.var_mean(z, dim=2, correction=0, keepdim=True)
            n = ((z - mean) * torch.rsqrt(var + EPS)).flatten(1) * weight + bias
            if case["gated"]:
                gate = st["gate"].detach()[cut].double().requires_grad_(True)
                leaves.append(gate)
                out = n * act(gate)
            else:
                out = act(n)
        outs.append(out.detach())
        if case["train"]:
            g = torch.autograd.grad(out, leaves, st["gy"][cut].double())
            gxs.append(g[0])
            sums = [sums[0] + g[1], sums[1] + g[2]]
            if case["gated"]:
                ggs.append(g[3])
    result = [torch.cat(outs)]
    if case["train"]:
        result.append(torch.cat(gxs))
        if case["gated"]:
            result.append(torch.cat(ggs))
        result += [t.detach() for t in sums]
    return result
