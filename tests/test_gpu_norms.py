"""Norms around a block on the GPU against plain implementations in 64 bits.

Bounds, from the arithmetic: a result of type t is rounded once (half a unit in
the last place, ``UNIT``). In fp32, a sum of n squares or products over the
threads of a row passes fewer than n / 32 + 16 additions, each off by at most
2^-24 of the magnitudes' sum, and is relative to a mean square that is of one
sign; the other steps of a value (products, the root, its reciprocal, the
additions) are fewer than 16. So a value is off by at most ``steps(n) * 2^-24``
of its terms' magnitudes."""

import math
import os
import subprocess
import sys

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L
from test_gpu_experts import TINY, TYPES, UNIT, gen, randn

pytestmark = pytest.mark.gpu

DEV = "cuda"
NAMES = ("x", "h", "norm_in", "norm_out", "gate")
L_CODE = {torch.float32: L.ES_F32, torch.bfloat16: L.ES_BF16, torch.float16: L.ES_F16}


def steps(n):
    return 2.0 ** -24 * (n / 32 + 48)


def make(g, T, D, dtype, gate, after, before, weights=None, scale=1.0):
    shape = {"channel": (D,), "row": (1, D), "token": (T, 1), "full": (T, D)}.get(gate)
    wt = weights or dtype
    return {"x": randn(g, T, D, dtype=dtype, scale=2.0 * scale), "h": randn(g, T, D, dtype=dtype, scale=0.5 * scale),
            "norm_in": randn(g, D, dtype=wt) if before else None, "norm_out": randn(g, D, dtype=wt) if after else None,
            "gate": randn(g, *shape, dtype=dtype) if gate else None}


def reference(v, scale, eps, dout=None, dy=None):
    """(values, magnitudes of their terms), by the formulas, in 64 bits."""
    d = {n: t.detach().double() for n, t in v.items() if t is not None}
    x, h = d["x"], d.get("h", torch.zeros_like(d["x"]))
    D = x.shape[1]
    gate = scale * d.get("gate", torch.ones((), dtype=torch.float64, device=DEV))
    r1 = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    hat = h * r1
    z = hat * d["norm_out"] if "norm_out" in d else h
    out = x + gate * z
    r2 = 1 / (out.square().mean(1, keepdim=True) + eps).sqrt()
    unit, big = out * r2, (x.abs() + (gate * z).abs())
    val, mag = {"out": out}, {"out": big}
    if "norm_in" in d:
        val["y"] = unit * d["norm_in"]
        # the mean of out^2 moves by twice the relative share of out's own error in its norm
        rel = (big.norm(dim=1, keepdim=True) / out.norm(dim=1, keepdim=True).clamp(min=1e-300))
        mag["y"] = (big * r2 + unit.abs() * (1 + rel)) * d["norm_in"].abs()
    if dout is None and dy is None:
        return val, mag
    back = dy.double() * d["norm_in"] if dy is not None else torch.zeros_like(x)
    do = dout.double() if dout is not None else torch.zeros_like(x)
    rel = 1 + (big.norm(dim=1, keepdim=True) / out.norm(dim=1, keepdim=True).clamp(min=1e-300))
    c2, m2 = (back * unit).mean(1, keepdim=True), (back * unit).abs().mean(1, keepdim=True)
    dx = do + r2 * (back - unit * c2)
    mdx = do.abs() + r2 * (back.abs() + big * r2 * m2) * rel
    dz, mdz = gate * dx, gate.abs() * mdx
    dh, mdh = dz, mdz
    if "norm_out" in d:
        b, mb = dz * d["norm_out"], mdz * d["norm_out"].abs()
        dh = r1 * (b - hat * (b * hat).mean(1, keepdim=True))
        mdh = r1 * (mb + hat.abs() * (mb * hat.abs()).mean(1, keepdim=True))
    val |= {"dx": dx, "dh": dh}
    mag |= {"dx": mdx, "dh": mdh}
    if "norm_in" in d:
        dy64 = dy.double() if dy is not None else torch.zeros_like(x)
        val["dnorm_in"], mag["dnorm_in"] = (dy64 * unit).sum(0), (dy64.abs() * big * r2 * rel).sum(0)
    if "norm_out" in d:
        val["dnorm_out"], mag["dnorm_out"] = (dz * hat).sum(0), (mdz * hat.abs()).sum(0)
    if "gate" in d:
        dg, mg = scale * z * dx, abs(scale) * z.abs() * mdx
        for dim in (0, 1):
            if d["gate"].dim() == 1 and dim == 0:
                dg, mg = dg.sum(0), mg.sum(0)
            elif d["gate"].dim() == 2 and d["gate"].shape[dim] == 1:
                dg, mg = dg.sum(dim, keepdim=True), mg.sum(dim, keepdim=True)
        val["dgate"], mag["dgate"] = dg, mg
    return val, mag


def close(name, got, ref, mag, n):
    assert got.shape == ref.shape, name
    bound = UNIT[got.dtype] * ref.abs() + steps(n) * mag + TINY[got.dtype]
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), (name, float((err - bound).max()))


def check(v, scale=0.7, eps=1e-6, grads=True, g=None, skip=None):
    T, D = v["x"].shape
    names = [n for n in NAMES if v.get(n) is not None]
    if grads:
        for n in names:
            v[n].requires_grad_()
    out, y = E.residual_norm(v["x"], v["h"], v["norm_in"], v["norm_out"], v["gate"], scale, eps)
    assert (y is None) == (v["norm_in"] is None)
    got = {"out": out} if y is None else {"out": out, "y": y}
    dout = dy = None
    if grads:
        dout = randn(g, T, D, dtype=out.dtype) if skip != "out" else None
        dy = randn(g, T, D, dtype=out.dtype) if y is not None and skip != "y" else None
        pairs = [(o, d) for o, d in ((out, dout), (y, dy)) if d is not None]
        for n, d in zip(names, torch.autograd.grad([p[0] for p in pairs], [v[n] for n in names], [p[1] for p in pairs])):
            got["d" + n] = d
            assert d.dtype == v[n].dtype
    val, mag = reference(v, scale, eps, dout, dy)
    assert set(got) == set(val)
    for n in got:
        close(n, got[n].detach(), val[n], mag[n], D + (T if n[:2] == "dn" or n == "dgate" else 0))
    E.check_device_errors()
    return got


@pytest.mark.parametrize("T,D", [(1, 1), (3, 8), (2, 7), (130, 64), (33, 264), (5, 1000), (9, 4096), (4, 5001),
                                 (3, 8200), (2, 16392), (2, 40000), (700, 48)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["", "channel", "token", "full"])
def test_residual_norm(T, D, dtype, gate):
    g = gen(T * D)
    check(make(g, T, D, dtype, gate, True, True), g=g)


@pytest.mark.parametrize("after,before", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["", "channel", "row", "token", "full"])
def test_residual_norm_parts(after, before, dtype, gate):
    g = gen(len(gate))
    for T, D in ((37, 520), (6, 33)):
        check(make(g, T, D, dtype, gate, after, before), g=g)
        check(make(g, T, D, dtype, gate, after, before), grads=False)


@pytest.mark.parametrize("skip", ["out", "y"])
def test_one_output_unused(skip):
    g = gen(5)
    for gate in ("", "channel", "token"):
        got = check(make(g, 21, 72, torch.float32, gate, True, True), g=g, skip=skip)
        if skip == "y":
            assert not got["dnorm_in"].any()


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_weights_in_fp32(dtype):
    g = gen(7)
    for T, D in ((50, 512), (11, 77)):
        check(make(g, T, D, dtype, "full", True, True, weights=torch.float32), g=g)


@pytest.mark.parametrize("T", [1, 295, 297, 4000])
def test_many_rows(T):
    """Column sums over more rows than groups walk them."""
    g = gen(T)
    for D in (96, 1032):
        check(make(g, T, D, torch.bfloat16, "channel", True, True), g=g)
        check(make(g, T, D, torch.float32, "channel", True, True), g=g)


@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm(dtype):
    g = gen(3)
    for T, D in ((1, 1), (40, 256), (7, 1001), (3, 33000)):
        x, w = randn(g, T, D, dtype=dtype).requires_grad_(), randn(g, D, dtype=dtype).requires_grad_()
        dy = randn(g, T, D, dtype=dtype)
        y = E.rms_norm(x, w, 1e-5)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        v = {"x": x, "norm_in": w}
        val, mag = reference(v, 0.0, 1e-5, None, dy)
        for n, t in (("y", y.detach()), ("dx", dx), ("dnorm_in", dw)):
            close(n, t, val[n], mag[n], D + T)
        with torch.no_grad():
            assert torch.equal(E.rms_norm(x, w, 1e-5), y)


def test_layouts():
    g = gen(11)
    T, D = 19, 264
    base = make(g, T, D, torch.bfloat16, "full", True, True)
    want = check({n: t.clone() for n, t in base.items()}, grads=False)

    def padded(t):
        wide = torch.zeros(T, D + 24, dtype=t.dtype, device=DEV)
        wide[:, 8:8 + D] = t
        return wide[:, 8:8 + D]

    def odd(t):
        wide = torch.zeros(T, D + 3, dtype=t.dtype, device=DEV)
        wide[:, 1:1 + D] = t
        return wide[:, 1:1 + D]

    for lay in (padded, odd, lambda t: t.t().contiguous().t(), lambda t: torch.cat([t, t])[T:]):
        v = {n: lay(t) if t.dim() == 2 else t for n, t in base.items()}
        got = check(v, grads=False)
        assert torch.equal(got["out"], want["out"])
        v = {n: t.detach().clone() for n, t in v.items()}
        check({n: lay(t) if t.dim() == 2 else t for n, t in v.items()}, g=gen(1))
    rows = {**base, "x": base["x"][:1].expand(T, D), "gate": base["gate"][:, :1].expand(T, D)}
    check({n: t.detach() for n, t in rows.items()}, grads=False)
    v = {**base, "gate": base["gate"][:, 3:4]}
    check(v, grads=False)


def test_broadcast_leaf():
    """A row that is every token's, and a weight that is both norms', get the sum of their gradients."""
    g = gen(13)
    T, D = 23, 40
    leaf, w = randn(g, 1, D).requires_grad_(), randn(g, D).requires_grad_()
    h, dout, dy = randn(g, T, D), randn(g, T, D), randn(g, T, D)
    out, y = E.residual_norm(leaf.expand(T, D), h, w, w)
    dl, dw = torch.autograd.grad((out, y), (leaf, w), (dout, dy))
    val, mag = reference({"x": leaf.detach().expand(T, D), "h": h, "norm_in": w, "norm_out": w}, 1.0, 1e-6, dout, dy)
    close("dx", dl, val["dx"].sum(0, keepdim=True), mag["dx"].sum(0, keepdim=True), D + 32 * T)
    close("dw", dw, val["dnorm_in"] + val["dnorm_out"], mag["dnorm_in"] + mag["dnorm_out"], D + T)


def test_gradient_by_differences():
    g = gen(17)
    T, D = 4, 24
    for gate in ("channel", "token", "full"):
        v = make(g, T, D, torch.float32, gate, True, True)
        dout, dy = randn(g, T, D), randn(g, T, D)
        for t in v.values():
            t.requires_grad_()
        out, y = E.residual_norm(*[v[n] for n in NAMES], 0.7, 1e-4)
        grads = dict(zip(NAMES, torch.autograd.grad((out, y), [v[n] for n in NAMES], (dout, dy))))

        def value(n, t):
            w = {**{k: s.detach() for k, s in v.items()}, n: t}
            o, y = E.residual_norm(*[w[k] for k in NAMES], 0.7, 1e-4)
            return (o.double() * dout).sum() + (y.double() * dy).sum()

        step = 2.0 ** -7
        for n in NAMES:
            way = randn(g, *v[n].shape)
            way = way / way.norm()
            base = v[n].detach()
            rise = (value(n, base + step * way) - value(n, base - step * way)) / (2 * step)
            # a third derivative within 2^7 of the outputs' scale, and 2^-22 of values that add up to about 2 T D
            assert abs(float(rise - (grads[n].double() * way).sum())) <= step ** 2 / 6 * 2.0 ** 7 * T + 2.0 ** -22 * 8 * T * D / step


def test_largest_and_smallest():
    """Rows whose squares overflow are normalised; rows of zeros and tiny rows are ruled by eps."""
    big = torch.finfo(torch.float32).max
    D = 96
    g = gen(19)
    x = torch.zeros(6, D, device=DEV)
    x[0], x[1], x[2], x[4], x[5] = big, 1e30, 1e-30, -1e25, 1e-4
    x[1, ::2] *= -1
    w = randn(g, D)
    for d in (D, 5):
        y = E.rms_norm(x[:, :d].contiguous(), w[:d].contiguous(), 1e-6)
        ref = x[:, :d].double()
        ref = ref / (ref.square().mean(1, keepdim=True) + 1e-6).sqrt() * w[:d].double()
        assert bool(((y.double() - ref).abs() <= 64 * 2.0 ** -24 * ref.abs() + 1e-38).all())
    zero = torch.zeros_like(x)
    out, y = E.residual_norm(zero, x, w, w)
    z = (x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()) * w.double()
    assert bool(((out.double() - z).abs() <= 64 * 2.0 ** -24 * z.abs() + 1e-38).all())
    xs = torch.zeros(3, D, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(E.rms_norm(xs, w, 1e-6), xs, torch.ones(3, D, device=DEV))
    assert bool(((dx.double() - 1e3 * w.double()).abs() <= 64 * 2.0 ** -24 * 1e3 * w.abs()).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_poisoned_rows_stay_alone(dtype):
    g = gen(23)
    T, D = 12, 136
    v = make(g, T, D, dtype, "full", True, True)
    clean = E.residual_norm(*[v[n] for n in NAMES])
    v["h"][3, 7], v["x"][5, 1], v["h"][8, 0] = math.nan, math.inf, -math.inf
    out, y = E.residual_norm(*[v[n] for n in NAMES])
    rest = [t for t in range(T) if t not in (3, 5, 8)]
    assert torch.equal(out[rest], clean[0][rest]) and torch.equal(y[rest], clean[1][rest])
    assert bool(out[3].isnan().all()) and bool(y[3].isnan().all())
    assert bool(out[5, 1].isposinf()) and bool(y[5, 1].isnan()) and not y[5, 2:].any()
    assert bool(out[8, 0].isnan())


def test_empty():
    for T, D in ((0, 8), (4, 0), (0, 0)):
        x = torch.zeros(T, D, device=DEV, requires_grad=True)
        w = torch.ones(D, device=DEV, requires_grad=True)
        out, y = E.residual_norm(x, x, w, w, w)
        assert out.shape == y.shape == (T, D)
        dx, dw = torch.autograd.grad((out, y), (x, w), (torch.ones_like(out), torch.ones_like(y)))
        assert dx.shape == (T, D) and dw.shape == (D,) and not dw.any()


def test_past_32_bits():
    T, D = 70001, 32768  # 2.3 billion values
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=DEV)
    g = gen(29)
    x[-3:] = randn(g, 3, D, dtype=torch.bfloat16)
    w = randn(g, D, dtype=torch.bfloat16)
    y = E.rms_norm(x, w)
    assert torch.equal(y[-3:], E.rms_norm(x[-3:].clone(), w))
    assert not y[:-3].any()


def test_same_bits_twice_streams_and_graph():
    g = gen(31)
    v = make(g, 900, 520, torch.bfloat16, "channel", True, True)
    for t in v.values():
        t.requires_grad_()
    dout, dy = (randn(g, 900, 520, dtype=torch.bfloat16) for _ in range(2))

    def step():
        o, y = E.residual_norm(*[v[n] for n in NAMES], 0.7)
        return (o.detach(), y.detach(), *torch.autograd.grad((o, y), [v[n] for n in NAMES], (dout, dy)))

    first, second = step(), step()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, third))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    with torch.no_grad():
        v["x"].mul_(0.5)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    for call in (lambda: E.residual_norm(x, x[:3]), lambda: E.residual_norm(x, x.bfloat16()),
                 lambda: E.residual_norm(x, x, w[:7]), lambda: E.residual_norm(x, x, gate=w[:4]),
                 lambda: E.residual_norm(x, x, gate=x[:, :2]), lambda: E.residual_norm(x, x, w, eps=0.0),
                 lambda: E.residual_norm(x[0], x[0]), lambda: E.rms_norm(x, w, math.nan), lambda: E.rms_norm(x, w.cpu())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: E.rms_norm(x.double(), w), lambda: E.rms_norm(x, w.bfloat16()), lambda: E.rms_norm(x, None),
                 lambda: E.residual_norm(x, None), lambda: E.residual_norm(x, x, gate=w.half()),
                 lambda: E.residual_norm(x.half(), x.half(), w.half(), w)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        y = E.rms_norm(x.requires_grad_(), w)
        d, = torch.autograd.grad(y.sum(), x, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("D", [269, 521, 1501, 5001])
@pytest.mark.parametrize("dtype", [t for t in TYPES if t != torch.float32])
@pytest.mark.parametrize("gate", ["", "token", "channel"])
def test_odd_rows_of_many(D, dtype, gate):
    """Enough odd rows for two pieces a thread: without a gate by channel, the
    forward pass walks them value by value, the backward pass by pieces."""
    g = gen(D)
    check(make(g, 601, D, dtype, gate, False, True), g=g)
    check(make(g, 601, D, dtype, gate, False, True), grads=False)


def test_sizes_at_the_shared_memory_limit():
    """Rows whose columns take a little less than 48 KB, each the first call of its kernel in a process: bf16 gradients of
    three and of two columns' sums, and odd rows forwards with their weights and gate in shared memory."""
    code = ("import test_gpu_norms as t, torch\n"
            "bf, f32 = torch.bfloat16, torch.float32\n"
            "for T, D, dtype, gate, weights, grads in ((1000, 1000, bf, 'channel', None, True), (40, 4032, f32, 'channel',"
            " None, True), (9, 6080, bf, '', f32, True), (5, 8101, bf, 'channel', None, False),"
            " (5, 6101, bf, '', f32, False), (6, 4032, bf, 'channel', None, True)):\n"
            "    g = t.gen(D)\n"
            "    t.check(t.make(g, T, D, dtype, gate, True, True, weights=weights), grads=grads, g=g)\n"
            "print('passed')\n")
    here = os.path.dirname(os.path.abspath(__file__))
    env = {**os.environ, "PYTHONPATH": os.pathsep.join([here, os.path.dirname(here)])}
    run = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and "passed" in run.stdout, run.stdout[-2000:] + run.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
def test_gate_by_token_of_no_channels(dtype):
    """A row without channels leaves the gate's gradient a sum of nothing."""
    T = 5
    for fill in (math.nan, 3.0):  # memory that the allocator hands out again
        torch.full((T, 1), fill, dtype=dtype, device=DEV)
        x, gate = torch.zeros(T, 0, dtype=dtype, device=DEV), torch.ones(T, 1, dtype=dtype, device=DEV).requires_grad_()
        out, _ = E.residual_norm(x, x, gate=gate)
        dgate, = torch.autograd.grad(out, gate, torch.ones_like(out))
        assert dgate.shape == (T, 1) and not dgate.any()


@pytest.mark.parametrize("D", [64, 1000, 77, 33000])
@pytest.mark.parametrize("dtype", TYPES)
def test_entry_point_takes_no_dy_for_zero(D, dtype):
    """A norm_in's gradient that is asked for without a dy is zero, and the others are as without it."""
    lib, T = L.lib(), 30
    g = gen(D)
    x, h, w, dout = (randn(g, *s, dtype=dtype, scale=1e3) for s in ((T, D), (T, D), (D,), (T, D)))
    code, stream = L_CODE[dtype], torch.cuda.current_stream().cuda_stream
    out, y, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(T, 2, device=DEV)
    head = (x.data_ptr(), D, h.data_ptr(), D, code, T, D, w.data_ptr(), w.data_ptr(), code, None, L.ES_GATE_NONE, 0, 0.7)
    assert lib.es_residual_norm(*head, 1e-6, out.data_ptr(), y.data_ptr(), stats.data_ptr(), stream) == L.ES_OK
    nbytes = lib.es_residual_norm_grad_workspace_size(code, T, D, 2)
    got = []
    for asked in (False, True):
        ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV)  # NaN
        dx, dh, dw_in, dw_out = (torch.full_like(t, math.nan) for t in (x, h, w, w))
        assert lib.es_residual_norm_grad(*head, stats.data_ptr(), dout.data_ptr(), D, None, 0, dx.data_ptr(),
                                         dh.data_ptr(), None, dw_in.data_ptr() if asked else None, dw_out.data_ptr(),
                                         ws.data_ptr(), nbytes, stream) == L.ES_OK
        got.append((dx, dh, dw_out))
        assert not asked or not bool(dw_in.any())
    assert all(torch.equal(a, b) and not bool(a.isnan().any()) for a, b in zip(*got))


def test_scale_that_wants_a_gradient():
    """The residual's scale is a number. A tensor that wants a gradient would lose it."""
    x, w = torch.ones(4, 8, device=DEV), torch.ones(8, device=DEV)
    s = torch.tensor(0.5, device=DEV, requires_grad=True)
    with pytest.raises(TypeError, match="scale"):
        E.residual_norm(x, x, w, scale=s)
    router, w_in, w_out = torch.zeros(8, 2, device=DEV), torch.zeros(2, 8, 16, device=DEV), torch.zeros(2, 8, 8, device=DEV)
    with pytest.raises(TypeError, match="scale"):
        E.expert_mlp(x, router, w_in, w_out, 1, activation="silu", scale=s)
    with pytest.raises(TypeError, match="scale"):
        E.expert_mlp(x, router, E.quantize_block_weights(w_in), E.quantize_block_weights(w_out), 1, scale=s)
    with torch.no_grad():
        out = E.residual_norm(x, x, scale=s)[0]
    assert torch.equal(out, E.residual_norm(x, x, scale=0.5)[0])
