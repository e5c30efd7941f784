"""Cases of the expert operators: routing, products grouped by expert, the weighted sum back to tokens, 8-bit products.

Each case is one call (or the pair of calls that belong together) as a program makes it. ``run`` computes it
either through ``einjax_b200`` (``own`` true) or in its plain form: elementary torch operations in 32 bits,
rounded once at the end. ``exact`` computes it from the definition in 64 bits.

Shared notation: T tokens, E experts, k choices a token, R = T k routed rows, in the order of their experts.
``offsets`` (E + 1) bounds each expert's rows, ``order`` (R) names the choice t * k + j behind each row and
``position`` (T, k) is its inverse; a choice of no expert (-1) has no row, and the rows past offsets[E] are empty.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MASKED_EVERY = 37  # with "masked": one token in so many is padding, whose logits are all masked; it has no expert


# ------------------------------------------------------------------ cases

def listed():
    return [
        # Routing: logits -> chosen experts and their weights -> row order of the experts.
        # One decode step of a small batch: all latency.
        {"name": "route_decode", "op": "route", "T": 8, "E": 64, "k": 8, "dtype": "f32", "renorm": True,
         "masked": False, "grad": False},
        # A ragged prompt with padding tokens, weights as shares of the softmax over all experts.
        {"name": "route_prompt", "op": "route", "T": 4099, "E": 60, "k": 4, "dtype": "bf16", "renorm": False,
         "masked": True, "grad": False},
        # A training step's tokens, with the gradient of the logits.
        {"name": "route_train", "op": "route", "T": 32768, "E": 128, "k": 8, "dtype": "f32", "renorm": True,
         "masked": False, "grad": True},
        # Products grouped by expert. Decode: a few tokens, bound by reading the experts' weights.
        {"name": "grouped_decode", "op": "grouped", "T": 8, "E": 16, "k": 2, "K": 2048, "N": 4096, "dtype": "bf16",
         "gather": True, "masked": False, "grad": False},
        # A ragged prompt over many small experts: about 70 rows an expert, no size a power of two.
        {"name": "grouped_prompt", "op": "grouped", "T": 1031, "E": 60, "k": 4, "K": 2048, "N": 2816, "dtype": "f16",
         "gather": True, "masked": True, "grad": False},
        # A training step of a few large experts: the product and both gradients.
        {"name": "grouped_train", "op": "grouped", "T": 8192, "E": 8, "k": 2, "K": 4096, "N": 8192, "dtype": "bf16",
         "gather": True, "masked": False, "grad": True},
        # Training in 32 bits, on rows that are grouped already, at sizes that fill no tile.
        {"name": "grouped_train_f32", "op": "grouped", "T": 1500, "E": 16, "k": 2, "K": 1000, "N": 2024,
         "dtype": "f32", "gather": False, "masked": False, "grad": True},
        # The weighted sum back to tokens: a decode step, and a training step (with padding) with both gradients.
        {"name": "combine_decode", "op": "combine", "T": 16, "E": 64, "k": 8, "D": 4096, "dtype": "bf16",
         "masked": False, "grad": False},
        {"name": "combine_train", "op": "combine", "T": 16384, "E": 64, "k": 4, "D": 4096, "dtype": "bf16",
         "masked": True, "grad": True},
        # 8-bit products of float tokens, which the call quantises, with weights that were quantised before.
        # A projection in a decode step; the same over a long ragged prompt; experts over a prompt.
        {"name": "int8_decode", "op": "int8", "T": 16, "E": 0, "k": 1, "K": 4096, "N": 4096, "dtype": "bf16",
         "masked": False},
        {"name": "int8_prompt", "op": "int8", "T": 8191, "E": 0, "k": 1, "K": 4096, "N": 8192, "dtype": "bf16",
         "masked": False},
        {"name": "int8_experts", "op": "int8", "T": 2050, "E": 64, "k": 8, "K": 2048, "N": 1408, "dtype": "bf16",
         "masked": False},
    ]


def _size(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "combine", "int8"])
    k = rng.randint(1, 8)
    E = _size(rng, 8, 128)
    c = {"op": op, "k": k, "masked": rng.random() < 0.5}
    if op == "route":
        return {**c, "T": _size(rng, 1, 32768), "E": E, "dtype": rng.choice(["f32", "f32", "bf16"]),
                "renorm": rng.random() < 0.5, "grad": rng.random() < 0.5}
    if op == "combine":
        return {**c, "T": _size(rng, 1, 65536 // k), "E": E, "D": _size(rng, 256, 4096, 8),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "grad": rng.random() < 0.5}
    c["K"] = _size(rng, 256, 4096, 8 if op == "grouped" else 16)
    c["N"] = _size(rng, 256, 4096 if op == "grouped" else 8192, 8)
    most = 2 ** 28 // (c["K"] * c["N"])  # experts, by the memory of their weights
    if op == "grouped":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return {**c, "T": _size(rng, 1, (4096 if dtype == "f32" else 16384) // k),
                "E": min(E, most // 2 if dtype == "f32" else most), "dtype": dtype, "gather": rng.random() < 0.5,
                "grad": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "f16"])
    if rng.random() < 0.5:
        return {**c, "T": _size(rng, 1, 8192), "E": 0, "k": 1, "masked": False, "dtype": dtype}
    return {**c, "T": _size(rng, 1, 16384 // k), "E": min(E, most), "dtype": dtype}


# ----------------------------------------------------------------- inputs

def _logits(c, g):
    """Router logits: tokens disagree, and some experts are liked better than others."""
    x = torch.randn(c["T"], c["E"], generator=g, device="cuda") * 1.5
    x += torch.randn(c["E"], generator=g, device="cuda") * 0.5
    return x


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


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    s = {"c": c}

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    if c["op"] == "route":
        x = _logits(c, g)
        if c["masked"]:  # padding tokens, and an expert in eight that each other token may not use
            x = x.masked_fill(torch.rand(c["T"], c["E"], generator=g, device="cuda") < 0.125, -math.inf)
            x[torch.arange(c["T"], device="cuda") % MASKED_EVERY == MASKED_EVERY - 1] = -math.inf
        s["logits"] = x.to(dt).requires_grad_(c["grad"])
        if c["grad"]:
            s["dweights"] = torch.randn(c["T"], c["k"], generator=g, device="cuda")
        return s

    if c["E"]:  # the routing that came before, and the largest expert's rows, which the plain form pads to
        top = torch.sort(_logits(c, g), dim=1, descending=True, stable=True)
        experts = top.indices[:, :c["k"]].int()
        if c["masked"]:
            experts[torch.arange(c["T"], device="cuda") % MASKED_EVERY == MASKED_EVERY - 1] = -1
        s["weights"] = torch.softmax(top.values[:, :c["k"]], dim=1)
        s["offsets"], s["order"], s["position"] = _layout(experts, c["E"])
        s["capacity"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    rows = c["T"] * c["k"]

    if c["op"] == "grouped":
        s["x"] = randn(c["T"] if c["gather"] else rows, c["K"])
        s["w"] = randn(c["E"], c["K"], c["N"], scale=c["K"] ** -0.5)
        if c["grad"]:
            s["x"].requires_grad_()
            s["w"].requires_grad_()
            s["dy"] = randn(rows, c["N"])
    elif c["op"] == "combine":
        s["y"] = randn(rows, c["D"])
        if c["grad"]:
            s["y"].requires_grad_()
            s["weights"].requires_grad_()
            s["dout"] = randn(c["T"], c["D"])
    else:  # int8: activations with a few loud channels, weights quantised to 8 bits for each output channel
        x = torch.randn(c["T"], c["K"], generator=g, device="cuda")
        x *= torch.where(torch.rand(c["K"], generator=g, device="cuda") < 0.01, 8.0, 1.0)
        s["x"] = x.to(dt)
        shape = (c["E"], c["N"], c["K"]) if c["E"] else (c["N"], c["K"])
        w = torch.randn(*shape, generator=g, device="cuda") * c["K"] ** -0.5
        s["wscale"] = w.abs().amax(-1) / 127
        s["wq"] = torch.round(w / s["wscale"][..., None]).to(torch.int8)
    return s


# -------------------------------------------------------------- own calls

def _run_own(s):
    import einjax_b200 as eb
    c = s["c"]
    op = c["op"]
    if op == "route":
        weights, experts = eb.route_experts(s["logits"], c["k"], renormalize=c["renorm"])
        plan = eb.plan_experts(experts, c["E"])
        out = {"weights": weights, "experts": experts, "offsets": plan.offsets, "order": plan.order,
               "position": plan.position}
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad(weights, s["logits"], s["dweights"])
        return out
    plan = eb.ExpertPlan(s["offsets"], s["order"], s["position"]) if c["E"] else None
    if op == "grouped":
        y = eb.grouped_matmul(s["x"], s["w"], plan, gather=c["gather"])
        if not c["grad"]:
            return y
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if op == "combine":
        out = eb.combine_experts(s["y"], s["weights"], plan)
        if not c["grad"]:
            return out
        dy, dweights = torch.autograd.grad(out, (s["y"], s["weights"]), s["dout"])
        return {"out": out, "dy": dy, "dweights": dweights}
    q, scale = eb.quantize_rows(s["x"])
    return eb.int8_matmul(q, scale, s["wq"], s["wscale"], plan, gather=plan is not None, out_dtype=s["x"].dtype)


# ------------------------------------------------------------ plain forms

def _plain_route(s):
    c, logits = s["c"], s["logits"].detach()
    x = logits.float()
    top = torch.sort(x, dim=1, descending=True, stable=True)
    value, experts = top.values[:, :c["k"]], top.indices[:, :c["k"]]
    there = value > -math.inf
    peak = torch.where(there[:, :1], value[:, :1], 0.0)
    e = torch.exp(value - peak)
    total = (e if c["renorm"] else torch.exp(x - peak)).sum(1, keepdim=True)
    weights = torch.where(there, e / total, 0.0)
    experts = torch.where(there, experts, -1).int()
    offsets, order, position = _layout(experts, c["E"])
    out = {"weights": weights, "experts": experts, "offsets": offsets, "order": order, "position": position}
    if c["grad"]:
        dot = (weights * s["dweights"]).sum(1, keepdim=True)
        p = torch.where(there[:, :1], torch.exp(x - peak) / total, 0.0)
        dlogits = torch.zeros_like(x) if c["renorm"] else -p * dot
        chosen = torch.where(experts < 0, 0, experts).long()
        part = weights * (s["dweights"] - dot) if c["renorm"] else weights * s["dweights"]
        dlogits.scatter_add_(1, chosen, torch.where(there, part, 0.0))
        out["dlogits"] = dlogits.to(logits.dtype)
    return out


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


def _plain_grouped(s):
    c, n = s["c"], s["c"]["T"] * s["c"]["k"]
    x, w = s["x"].detach(), s["w"].detach()
    dt = x.dtype
    place, held = _padded_rows(s)
    xr = x.float()[torch.clamp(s["order"].long(), min=0) // c["k"]] if c["gather"] else x.float()
    xp, wf = _pad(xr, place, held), w.float()
    y = _unpad(torch.bmm(xp, wf), place, held, n).to(dt)
    if not c["grad"]:
        return y
    dp = _pad(s["dy"].float(), place, held)
    dw = torch.bmm(xp.transpose(1, 2), dp).to(dt)
    dx = _unpad(torch.bmm(dp, wf.transpose(1, 2)), place, held, n)
    if c["gather"]:
        at = s["position"].long()
        dx = torch.where(at[..., None] >= 0, dx[torch.clamp(at, min=0)], 0.0).sum(1)
    return {"y": y, "dx": dx.to(dt), "dw": dw}


def _plain_combine(s):
    c, dt = s["c"], s["y"].dtype
    y, weights = s["y"].detach().float(), s["weights"].detach()
    at = s["position"].long()
    picked = torch.where(at[..., None] >= 0, y[torch.clamp(at, min=0)], 0.0)
    out = (picked * weights[..., None]).sum(1).to(dt)
    if not c["grad"]:
        return out
    dout = s["dout"].float()
    dweights = (picked * dout[:, None, :]).sum(2)
    choice = s["order"].long()
    token = torch.clamp(choice, min=0) // c["k"]
    share = torch.where(choice >= 0, weights.reshape(-1)[torch.clamp(choice, min=0)], 0.0)
    return {"out": out, "dy": (dout[token] * share[:, None]).to(dt), "dweights": dweights}


def _plain_int8(s):
    c, dt = s["c"], s["x"].dtype
    x = s["x"].float()
    scale = x.abs().amax(1) / 127
    q = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), 0.0)
    if not c["E"]:
        y = q @ s["wq"].float().t()
        return (y * scale[:, None] * s["wscale"]).to(dt)
    token = torch.clamp(s["order"].long(), min=0) // c["k"]
    place, held = _padded_rows(s)
    y = torch.bmm(_pad(q[token], place, held), s["wq"].float().transpose(1, 2))
    y = y * _pad(scale[token][:, None], place, held) * s["wscale"][:, None, :]
    return _unpad(y, place, held, c["T"] * c["k"]).to(dt)


PLAIN = {"route": _plain_route, "grouped": _plain_grouped, "combine": _plain_combine, "int8": _plain_int8}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return PLAIN[state["c"]["op"]](state)


# ---------------------------------------------------- floors and 64 bits

def _used(c):
    """Experts that a step of T tokens reads, on average, were each choice as likely."""
    return c["E"] * (1 - (1 - min(c["k"], c["E"]) / c["E"]) ** c["T"])


def work(case):
    c = case
    b, T, k, E = BYTES[c["dtype"]], c["T"], c["k"], c["E"]
    R = T * k
    if c["op"] == "route":  # logits in; weights, experts, order, position and offsets out
        n = T * E * b + R * 16 + (E + 1) * 4
        return {"bytes": n + (T * E * b + R * 4 if c["grad"] else 0), "flops": T * E * 4}
    if c["op"] == "combine":  # each row in, each token out, and the weights and places of the choices
        n = R * c["D"] * b + T * c["D"] * b + R * 8
        return {"bytes": n + ((R + T) * c["D"] * b + R * 8 if c["grad"] else 0),
                "flops": 2 * R * c["D"] * (3 if c["grad"] else 1)}
    K, N = c["K"], c["N"]
    if c["op"] == "grouped":
        xin = T if c["gather"] else R
        n = xin * K * b + _used(c) * K * N * b + R * N * b + (R + E) * 4
        if c["grad"]:
            n += R * N * b + xin * K * b + E * K * N * b
        return {"bytes": n, "flops": 2 * R * K * N * (3 if c["grad"] else 1)}
    used = _used(c) if E else 1
    return {"bytes": T * K * b + used * (K * N + 4 * N) + R * N * b, "flops": 2 * R * K * N}


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    with torch.no_grad():
        if c["op"] == "route":
            return _exact_route(c, s)
        if c["op"] == "combine":
            return _exact_combine(c, s)
        return _exact_grouped(c, s) if c["op"] == "grouped" else _exact_int8(c, s)


def _exact_route(c, s):
    x = s["logits"].detach().double()
    T, k = c["T"], c["k"]
    rest, rows = x.clone(), torch.arange(T, device=x.device)
    experts = torch.full((T, k), -1, dtype=torch.int64, device=x.device)
    for j in range(k):  # the largest that is left, the lowest index of equals
        best = rest.amax(1)
        at = (rest == best[:, None]).int().argmax(1)
        experts[:, j] = torch.where(best > -math.inf, at, -1)
        rest[rows, at] = -math.inf
    chosen = torch.zeros_like(x, dtype=torch.bool)
    for j in range(k):
        live = experts[:, j] >= 0
        chosen[rows[live], experts[live, j]] = True
    over = chosen if c["renorm"] else x > -math.inf
    p = torch.softmax(torch.where(over, x, -math.inf), dim=1).nan_to_num(0.0)
    at = experts.clamp(min=0)
    weights = torch.where(experts >= 0, p.gather(1, at), 0.0)
    out = {"weights": weights, "experts": None, "offsets": None, "order": None, "position": None}
    if c["grad"]:
        g = torch.zeros_like(x)
        for j in range(k):
            live = experts[:, j] >= 0
            g[rows[live], experts[live, j]] = s["dweights"].double()[live, j]
        out["dlogits"] = p * (g - (p * g).sum(1, keepdim=True))
    return out


def _exact_rows(c, s):
    """Each expert's rows and their tokens, on the host."""
    off, order = s["offsets"].tolist(), s["order"].long()
    for e in range(c["E"]):
        if off[e] < off[e + 1]:
            rows = slice(off[e], off[e + 1])
            yield e, rows, order[rows] // c["k"]


def _exact_grouped(c, s):
    x, w = s["x"].detach().double(), s["w"].detach()
    n = c["T"] * c["k"]
    y = x.new_zeros(n, c["N"])
    dx, dw = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=x.device) if c["grad"] else None
    for e, rows, tokens in _exact_rows(c, s):
        xe, we = x[tokens] if c["gather"] else x[rows], w[e].double()
        y[rows] = xe @ we
        if c["grad"]:
            g = s["dy"][rows].double()
            dw[e] = xe.t() @ g
            back = g @ we.t()
            if c["gather"]:
                dx.index_add_(0, tokens, back)
            else:
                dx[rows] = back
    return {"y": y, "dx": dx, "dw": dw} if c["grad"] else y


def _exact_combine(c, s):
    y, weights = s["y"].detach().double(), s["weights"].detach().double()
    out = y.new_zeros(c["T"], c["D"])
    dy, dweights = torch.zeros_like(y), torch.zeros_like(weights)
    for j in range(c["k"]):
        at = s["position"][:, j].long()
        live = at >= 0
        out[live] += weights[live, j, None] * y[at[live]]
        if c["grad"]:
            dout = s["dout"][live].double()
            dy[at[live]] = weights[live, j, None] * dout
            dweights[live, j] = (dout * y[at[live]]).sum(1)
    return {"out": out, "dy": dy, "dweights": dweights} if c["grad"] else out


def _exact_int8(c, s):
    """The definition holds the tokens' scales in 32 bits and their values in 8: both are rounded here too."""
    x = s["x"].double()
    scale = (x.abs().amax(1) / 127).float().double()
    q = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), 0.0).clamp(-127, 127)
    wq, wscale = s["wq"], s["wscale"].double()
    if not c["E"]:
        return (q @ wq.double().t()) * scale[:, None] * wscale
    y = x.new_zeros(c["T"] * c["k"], c["N"])
    for e, rows, tokens in _exact_rows(c, s):
        y[rows] = (q[tokens] @ wq[e].double().t()) * scale[tokens, None] * wscale[e]
    return y
