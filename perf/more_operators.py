"""Cases of the gated products, the 8-bit floating-point products and the norms around a block.

Each case is one call (or the calls that belong together) as a program makes it. ``run`` computes it either
through ``einjax_b200`` (``own`` true) or in its plain form: elementary torch operations in 32 bits, rounded
once at the end. ``exact`` computes it from the definition in 64 bits.

gated   h[r] = act(x[r] @ gate) * (x[r] @ up), with w = [gate | up]: dense (E = 0), or by expert
fp8     y[r] = x[r] @ w^T with both in e4m3, x with a scale for each 128 values of a row, w for each 128 x 128;
        with an activation x is act(g) * u of the row's two halves, rounded to 8 bits as it is made
norm    out = x + scale * gate * (rms(h) * norm_out), y = rms(out) * norm_in

Shared notation: T tokens, E experts, k choices a token, R = T k routed rows, in the order of their experts.
``offsets`` (E + 1) bounds each expert's rows, ``order`` (R) names the choice t * k + j behind each row and
``position`` (T, k) is its inverse; a choice of no expert (-1) has no row, and the rows past offsets[E] are empty.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128        # values that share a scale
MASKED_EVERY = 37  # with "masked": one token in so many is padding and has no expert
EPS = 1e-6
SCALE = 0.7        # of the residual


# ------------------------------------------------------------------ cases

def listed():
    return [
        # Gate, up, activation and product. One decode step of a small batch over a few experts: reading weights.
        {"name": "gated_decode", "op": "gated", "T": 8, "E": 16, "k": 2, "K": 2048, "F": 2048, "dtype": "bf16",
         "act": "silu", "gather": True, "masked": False, "grad": False},
        # A ragged prompt with padding over many small experts.
        {"name": "gated_prompt", "op": "gated", "T": 1031, "E": 60, "k": 4, "K": 2048, "F": 1408, "dtype": "f16",
         "act": "silu", "gather": True, "masked": True, "grad": False},
        # A training step of a dense block: the product and both gradients.
        {"name": "gated_train", "op": "gated", "T": 8192, "E": 0, "k": 1, "K": 4096, "F": 8192, "dtype": "bf16",
         "act": "gelu_tanh", "gather": False, "masked": False, "grad": True},
        # Training in 32 bits by expert, on rows that are grouped already, at sizes that fill no tile.
        {"name": "gated_train_f32", "op": "gated", "T": 1500, "E": 16, "k": 2, "K": 1000, "F": 1012, "dtype": "f32",
         "act": "gelu", "gather": False, "masked": False, "grad": True},
        # 8-bit products of float tokens, which the call rounds, with weights that were rounded before.
        # A projection in a decode step; the same over a long ragged prompt; experts over a prompt, into the
        # gated block and out of it (where the activation is part of the rounding).
        {"name": "fp8_decode", "op": "fp8", "T": 16, "E": 0, "k": 1, "K": 4096, "N": 4096, "dtype": "bf16",
         "act": "", "masked": False},
        {"name": "fp8_prompt", "op": "fp8", "T": 8191, "E": 0, "k": 1, "K": 4096, "N": 8192, "dtype": "bf16",
         "act": "", "masked": False},
        {"name": "fp8_experts_in", "op": "fp8", "T": 2050, "E": 64, "k": 8, "K": 2048, "N": 2816, "dtype": "bf16",
         "act": "", "masked": True},
        {"name": "fp8_experts_out", "op": "fp8", "T": 2050, "E": 64, "k": 8, "K": 1408, "N": 2048, "dtype": "bf16",
         "act": "silu", "masked": False},
        # Norms around a block. A decode step; a prompt of odd width whose block is gated by token and has no
        # norm of its own; a training step with both gradients and a gate by channel; the same in 32 bits with
        # a gate of its own for every value.
        {"name": "norm_decode", "op": "norm", "T": 16, "D": 4096, "dtype": "bf16", "gate": "", "after": True,
         "before": True, "grad": False},
        {"name": "norm_prompt", "op": "norm", "T": 4099, "D": 5001, "dtype": "f16", "gate": "token", "after": False,
         "before": True, "grad": False},
        {"name": "norm_train", "op": "norm", "T": 16384, "D": 4096, "dtype": "bf16", "gate": "channel",
         "after": True, "before": True, "grad": True},
        {"name": "norm_train_f32", "op": "norm", "T": 5000, "D": 1544, "dtype": "f32", "gate": "full", "after": True,
         "before": True, "grad": True},
    ]


def _size(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["gated", "fp8", "norm"])
    if op == "norm":
        step = rng.choice([8, 8, 8, 1])
        D = _size(rng, 64, 16384, step)
        return {"op": op, "T": _size(rng, 1, 2 ** 26 // D), "D": D, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "gate": rng.choice(["", "channel", "token", "full"]), "after": rng.random() < 0.7,
                "before": rng.random() < 0.7, "grad": rng.random() < 0.5}
    step = rng.choice([16, 16, 8, 1])
    E = rng.choice([0, _size(rng, 2, 128)])
    k = rng.randint(1, min(E, 8)) if E else 1
    c = {"op": op, "E": E, "k": k, "K": _size(rng, 128, 4096, step), "masked": E > 0 and rng.random() < 0.5}
    if op == "gated":
        c["F"] = _size(rng, 128, 4096, step)
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        few = c["dtype"] == "f32"
        c["E"] = min(E, 2 ** (27 if few else 28) // (2 * c["K"] * c["F"]))  # by the memory of the weights
        c["k"] = min(k, c["E"]) if E else 1
        return {**c, "T": _size(rng, 1, (4096 if few else 16384) // c["k"]), "grad": rng.random() < 0.5,
                "gather": E > 0 and rng.random() < 0.5, "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])}
    c["N"] = _size(rng, 128, 8192, step)
    c["E"] = min(E, 2 ** 28 // (c["K"] * c["N"]))
    c["k"] = min(k, c["E"]) if E else 1
    return {**c, "T": _size(rng, 1, 16384 // c["k"]), "dtype": rng.choice(["bf16", "f16"]),
            "act": rng.choice(["", "", "silu", "gelu_tanh"])}


# ----------------------------------------------------------------- inputs

def _layout(experts, E):
    """(offsets, order, position) of the chosen experts, int32; -1 is no expert."""
    T, k = experts.shape
    key = torch.where(experts < 0, E, experts).reshape(-1).long()
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(E, device=key.device)[None, :]).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    rows = torch.arange(T * k, device=key.device)
    kept = rows < offsets[E]
    position = torch.empty_like(order)
    position[order] = torch.where(kept, rows, -1)
    return offsets.int(), torch.where(kept, order, -1).int(), position.reshape(T, k).int()


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    s = {"c": c}

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    if c["op"] == "norm":
        T, D = c["T"], c["D"]
        loud = 1 + 4 * (torch.rand(D, generator=g, device="cuda") < 0.01)  # a residual stream has a few loud channels
        s["x"], s["h"] = (randn(T, D, scale=2.0) * loud).to(dt), randn(T, D, scale=0.5).to(dt)
        s["norm_out"] = (1 + randn(D, scale=0.2)).to(dt) if c["after"] else None
        s["norm_in"] = (1 + randn(D, scale=0.2)).to(dt) if c["before"] else None
        shape = {"channel": (D,), "token": (T, 1), "full": (T, D)}.get(c["gate"])
        s["gate"] = torch.sigmoid(randn(*shape)).to(dt) if shape else None
        if c["grad"]:
            for name in ("x", "h", "gate", "norm_out", "norm_in"):
                if s[name] is not None:
                    s[name].requires_grad_()
            s["dout"] = randn(T, D).to(dt)
            s["dy"] = randn(T, D).to(dt) if c["before"] else None
        return s

    T, E, k, K = c["T"], c["E"], c["k"], c["K"]
    if E:  # the routing that came before, and the largest expert's rows, which the plain form pads to
        logits = randn(T, E, scale=1.5) + randn(E, scale=0.5)
        experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].int()
        if c["masked"]:
            experts[torch.arange(T, device="cuda") % MASKED_EVERY == MASKED_EVERY - 1] = -1
        s["offsets"], s["order"], s["position"] = _layout(experts, E)
        s["capacity"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())

    if c["op"] == "gated":
        s["x"] = randn(T if c["gather"] else T * k, K).to(dt)
        s["w"] = randn(*((E, K, 2 * c["F"]) if E else (K, 2 * c["F"])), scale=K ** -0.5).to(dt)
        if c["grad"]:
            s["x"].requires_grad_()
            s["w"].requires_grad_()
            s["dh"] = randn(T * k, c["F"]).to(dt)
        return s

    # activations with a few loud channels, by token, or with an activation by grouped row
    x = randn(T * k if c["act"] else T, 2 * K if c["act"] else K)
    x *= torch.where(torch.rand(x.shape[1], generator=g, device="cuda") < 0.01, 8.0, 1.0)
    s["x"] = x.to(dt)
    w = randn(max(E, 1), c["N"], K, scale=K ** -0.5)
    padded = torch.nn.functional.pad(w, (0, -K % BLOCK, 0, -c["N"] % BLOCK))
    peak = padded.reshape(w.shape[0], _blocks(c["N"]), BLOCK, _blocks(K), BLOCK).abs().amax((2, 4))
    ws = peak / 448
    wq = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device="cuda")
    for e in range(w.shape[0]):
        wq[e] = (w[e] / _spread(ws[e], c["N"], K)).to(torch.float8_e4m3fn)
    s["wq"], s["wscale"] = (wq, ws) if E else (wq[0], ws[0])
    return s


def _spread(scale, n, k):
    """A scale for each BLOCK x BLOCK block -> one for each value."""
    return scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


# -------------------------------------------------------------- own calls

def _run_own(s):
    import einjax_b200 as eb
    c = s["c"]
    if c["op"] == "norm":
        out, y = eb.residual_norm(s["x"], s["h"], norm_in=s["norm_in"], norm_out=s["norm_out"], gate=s["gate"],
                                  scale=SCALE, eps=EPS)
        got = {"out": out} if y is None else {"out": out, "y": y}
        if c["grad"]:
            names = [n for n in ("x", "h", "gate", "norm_out", "norm_in") if s[n] is not None]
            outs, grads = ((out,), (s["dout"],)) if y is None else ((out, y), (s["dout"], s["dy"]))
            for n, d in zip(names, torch.autograd.grad(outs, [s[n] for n in names], grads)):
                got["d" + n] = d
        return got
    plan = eb.ExpertPlan(s["offsets"], s["order"], s["position"]) if c["E"] else None
    if c["op"] == "gated":
        h = eb.gated_matmul(s["x"], s["w"], plan, gather=c["gather"], activation=c["act"])
        if not c["grad"]:
            return h
        dx, dw = torch.autograd.grad(h, (s["x"], s["w"]), s["dh"])
        return {"h": h, "dx": dx, "dw": dw}
    q, scale = eb.quantize_blocks(s["x"], activation=c["act"] or None)
    return eb.fp8_matmul(q, scale, s["wq"], s["wscale"], plan, gather=plan is not None and not c["act"],
                         out_dtype=s["x"].dtype)


# ------------------------------------------------------------ plain forms

def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)
    return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)


def _plain_norm(s):
    c, dt = s["c"], s["x"].dtype
    x, h = s["x"].detach().float(), s["h"].detach().float()
    z, hat, r1 = h, None, None
    if c["after"]:
        r1 = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
        hat = h * r1
        z = hat * s["norm_out"].detach().float()
    gate = s["gate"].detach().float() if c["gate"] else torch.ones((), device=x.device)
    out = x + SCALE * gate * z
    got = {"out": out.to(dt)}
    if c["before"]:
        r2 = torch.rsqrt((out * out).mean(1, keepdim=True) + EPS)
        unit = out * r2
        got["y"] = (unit * s["norm_in"].detach().float()).to(dt)
    if not c["grad"]:
        return got
    d = s["dout"].float()
    if c["before"]:
        dy = s["dy"].float()
        back = dy * s["norm_in"].detach().float()
        d = d + r2 * (back - unit * (back * unit).mean(1, keepdim=True))
    got["dx"] = d.to(dt)
    dz = SCALE * gate * d
    dh = dz
    if c["after"]:
        back = dz * s["norm_out"].detach().float()
        dh = r1 * (back - hat * (back * hat).mean(1, keepdim=True))
    got["dh"] = dh.to(dt)
    if c["gate"]:
        dg = SCALE * z * d
        got["dgate"] = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True),
                        "full": lambda: dg}[c["gate"]]().to(dt)
    if c["after"]:
        got["dnorm_out"] = (dz * hat).sum(0).to(dt)
    if c["before"]:
        got["dnorm_in"] = (dy * unit).sum(0).to(dt)
    return got


def _padded_rows(s):
    """(E, capacity) row of each padded place, and whether it holds one."""
    off = s["offsets"].long()
    at = torch.arange(s["capacity"], device=off.device)[None, :]
    row = off[:-1, None] + at
    held = row < off[1:, None]
    return torch.where(held, row, 0), held


def _pad(rows, place, held):
    return torch.where(held[..., None], rows[place], 0.0)


def _unpad(padded, place, held, n):
    out = padded.new_zeros(n, padded.shape[2])
    out[place[held]] = padded[held]
    return out


def _plain_gated(s):
    c, x, w = s["c"], s["x"].detach(), s["w"].detach().float()
    n, F, dt = c["T"] * c["k"], c["F"], s["x"].dtype
    xr = x.float()
    if c["E"]:
        place, held = _padded_rows(s)
        if c["gather"]:
            xr = xr[torch.clamp(s["order"].long(), min=0) // c["k"]]
        xr = _pad(xr, place, held)
    y = torch.matmul(xr, w)
    a, slope = _act(c["act"], y[..., :F])
    h = a * y[..., F:]
    if c["E"]:
        h = _unpad(h, place, held, n)
    if not c["grad"]:
        return h.to(dt)
    dh = s["dh"].float()
    if c["E"]:
        dh = _pad(dh, place, held)
    dy = torch.cat([dh * y[..., F:] * slope, dh * a], -1)
    dw = torch.matmul(xr.transpose(-1, -2), dy)
    dx = torch.matmul(dy, w.transpose(-1, -2))
    if c["E"]:
        dx = _unpad(dx, place, held, n)
        if c["gather"]:
            at = s["position"].long()
            dx = torch.where(at[..., None] >= 0, dx[torch.clamp(at, min=0)], 0.0).sum(1)
    return {"h": h.to(dt), "dx": dx.to(dt), "dw": dw.to(dt)}


def _rounded(x):
    """Values (rows, width) rounded to e4m3 with the smallest power of two as the scale of each BLOCK of a row
    that keeps them within 448, as the values they stand for."""
    rows, width = x.shape
    b = torch.nn.functional.pad(x, (0, -width % BLOCK)).reshape(rows, -1, BLOCK)
    peak = b.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(peak)  # 448 = 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(peak), torch.clamp(exponent - 9 + (mantissa > 0.875).int(), min=-126))
    q = (b / scale).to(torch.float8_e4m3fn).float() * scale
    return q.reshape(rows, -1)[:, :width]


def _plain_fp8(s):
    c, dt = s["c"], s["x"].dtype
    x = s["x"].float()
    if c["act"]:
        x = _act(c["act"], x[:, :c["K"]])[0] * x[:, c["K"]:]
    x = _rounded(x)
    w = s["wq"].float() * _spread(s["wscale"], c["N"], c["K"])
    if not c["E"]:
        return (x @ w.t()).to(dt)
    if not c["act"]:
        x = x[torch.clamp(s["order"].long(), min=0) // c["k"]]
    place, held = _padded_rows(s)
    y = torch.bmm(_pad(x, place, held), w.transpose(1, 2))
    return _unpad(y, place, held, c["T"] * c["k"]).to(dt)


PLAIN = {"gated": _plain_gated, "fp8": _plain_fp8, "norm": _plain_norm}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return PLAIN[state["c"]["op"]](state)


# ---------------------------------------------------- floors and 64 bits

def _used(c):
    """Experts that a step of T tokens reads, on average, were each choice as likely."""
    return c["E"] * (1 - (1 - min(c["k"], c["E"]) / c["E"]) ** c["T"]) if c["E"] else 1


def work(case):
    c = case
    b, T = BYTES[c["dtype"]], c["T"]
    if c["op"] == "norm":
        D = c["D"]
        gate = {"": 0, "channel": D, "token": T, "full": T * D}[c["gate"]]
        norms = D * (c["after"] + c["before"])
        n = 2 * T * D + (1 + c["before"]) * T * D + gate + norms
        if c["grad"]:
            n += (1 + c["before"]) * T * D + 2 * T * D + gate + norms
        return {"bytes": n * b, "flops": T * D * (20 if c["grad"] else 8)}
    E, K, R = c["E"], c["K"], T * c["k"]
    if c["op"] == "gated":
        F, xin = c["F"], T if c["gather"] else R
        n = xin * K * b + _used(c) * K * 2 * F * b + R * F * b + (R + E) * 4 * (E > 0)
        if c["grad"]:
            n += R * F * b + xin * K * b + max(E, 1) * K * 2 * F * b
        return {"bytes": n, "flops": 4 * R * K * F * (3 if c["grad"] else 1)}
    N = c["N"]
    xin = R * 2 * K if c["act"] else T * K
    return {"bytes": xin * b + _used(c) * (N * K + 4 * _blocks(N) * _blocks(K)) + R * N * b, "flops": 2 * R * K * N}


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "norm":
        return _exact_norm(c, s)
    with torch.no_grad():
        return _exact_gated(c, s) if c["op"] == "gated" else _exact_fp8(c, s)


def _exact_norm(c, s):
    names = [n for n in ("x", "h", "gate", "norm_out", "norm_in") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(c["grad"]) for n in names}

    def rms(t):
        return t / torch.sqrt(t.square().sum(1, keepdim=True) / c["D"] + EPS)

    block = rms(v["h"]) * v["norm_out"] if c["after"] else v["h"]
    if c["gate"]:
        block = block * v["gate"]
    out = v["x"] + block * SCALE
    got = {"out": out}
    if c["before"]:
        got["y"] = rms(out) * v["norm_in"]
    if c["grad"]:
        loss = (out * s["dout"].double()).sum()
        if c["before"]:
            loss = loss + (got["y"] * s["dy"].double()).sum()
        for n, d in zip(names, torch.autograd.grad(loss, [v[n] for n in names])):
            got["d" + n] = d
    return {n: t.detach() for n, t in got.items()}


def _exact_act(name, g):
    if name == "silu":
        return g * torch.special.expit(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    if name == "gelu_tanh":  # (1 + tanh a) / 2 = 1 / (1 + exp(-2 a))
        return g * torch.special.expit(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))
    return torch.relu(g)


def _exact_slope(name, g):
    if name == "silu":
        p = torch.special.expit(g)
        return p + g * p * torch.special.expit(-g)
    if name == "gelu":
        return torch.special.ndtr(g) + g * torch.exp(-g * g / 2) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        b = math.sqrt(8 / math.pi)
        a = b * (g + 0.044715 * g ** 3)
        p = torch.special.expit(a)
        return p + g * p * torch.special.expit(-a) * b * (1 + 0.134145 * g * g)
    return torch.where(g > 0, 1.0, 0.0)


def _groups(c, s):
    """Each expert (None: the dense matrix), its rows and the rows of x behind them."""
    if not c["E"]:
        yield None, slice(0, c["T"]), slice(0, c["T"])
        return
    off = s["offsets"].tolist()
    for e in range(c["E"]):
        if off[e] < off[e + 1]:
            rows = slice(off[e], off[e + 1])
            yield e, rows, s["order"][rows].long() // c["k"]


def _exact_gated(c, s):
    x, w, F = s["x"].detach().double(), s["w"].detach(), c["F"]
    h = x.new_zeros(c["T"] * c["k"], F)
    dx = torch.zeros_like(x)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device) if c["grad"] else None
    for e, rows, tokens in _groups(c, s):
        xe, we = x[tokens] if c["gather"] else x[rows], (w if e is None else w[e]).double()
        g, u = xe @ we[:, :F], xe @ we[:, F:]
        h[rows] = _exact_act(c["act"], g) * u
        if c["grad"]:
            d = s["dh"][rows].double()
            dg, du = d * u * _exact_slope(c["act"], g), d * _exact_act(c["act"], g)
            part = dw if e is None else dw[e]
            part[:, :F], part[:, F:] = xe.t() @ dg, xe.t() @ du
            back = dg @ we[:, :F].t() + du @ we[:, F:].t()
            if c["gather"]:
                dx.index_add_(0, tokens, back)
            else:
                dx[rows] = back
    return {"h": h, "dx": dx, "dw": dw} if c["grad"] else h


def _exact_fp8(c, s):
    """The definition holds x in 8 bits with a power of two for each block: both are rounded here too."""
    x, K = s["x"].double(), c["K"]
    if c["act"]:
        x = _exact_act(c["act"], x[:, :K]) * x[:, K:]
    for b in range(0, K, BLOCK):
        v = x[:, b:b + BLOCK]
        peak = v.abs().amax(1, keepdim=True)
        power = torch.where(peak > 0, torch.ceil(torch.log2(torch.clamp(peak, min=1e-300) / 448)), -126.0)
        power = torch.where(torch.exp2(power - 1) * 448 >= peak, power - 1, power)  # the logarithm's own rounding
        power = torch.where(torch.exp2(power) * 448 < peak, power + 1, power).clamp(min=-126)
        v = v * torch.exp2(-power)
        step = torch.exp2(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -6))) - 3)  # eight to a power of two
        x[:, b:b + BLOCK] = torch.round(v / step) * step * torch.exp2(power)
    y = x.new_zeros(c["T"] * c["k"], c["N"])
    for e, rows, tokens in _groups(c, s):
        wq, ws = (s["wq"], s["wscale"]) if e is None else (s["wq"][e], s["wscale"][e])
        w = wq.float().double() * _spread(ws.double(), c["N"], K)
        xe = x[rows] if c["act"] or e is None else x[tokens]
        y[rows] = xe @ w.t()
    return y
