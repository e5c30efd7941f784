"""Gated products on the GPU against plain implementations in 64 bits.

Bounds, from the arithmetic: each product g = x gate, u = x up is off by at most
``K * 2**-23`` of its terms' magnitudes (as in ``test_gpu_experts``), which reaches h
through slopes that are at most 1.13 (the derivative of every activation here) times
|u|, and |act|. The activation itself is off by a few units of fp32 and by its
argument's rounding, which its tail multiplies: by |g| for exp(-g), g^2 for erfc, and
the cubic's own size for tanh's (``act_error``). h is rounded once. The slopes are
rounded once, their products with dh once more, and the gradients once: dx and dw are
within those roundings of their terms, the sums' error beside them."""

import math

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L
from test_gpu_experts import SIZES, TINY, TYPES, UNIT, gen, make_plan, randn

pytestmark = pytest.mark.gpu

DEV = "cuda"
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def act_ref(name, g):
    """act and act' in 64 bits."""
    if name == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * torch.sigmoid(-g))
    if name == "gelu":
        p = torch.special.erfc(-g / math.sqrt(2)) / 2
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        b = math.sqrt(8 / math.pi)
        p = torch.sigmoid(b * (g + 0.044715 * g ** 3))
        return g * p, p + g * p * torch.sigmoid(-b * (g + 0.044715 * g ** 3)) * b * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).double()


def act_error(g):
    return 2.0 ** -22 * (4 + g.abs() + g * g + g.abs() ** 3 / 4)


def groups(plan, gather, x):
    if plan is None:
        yield slice(None), slice(0, x.shape[0]), torch.arange(x.shape[0], device=DEV)
        return
    off, order = plan.offsets.tolist(), plan.order.long()
    for e in range(plan.num_experts):
        r = slice(off[e], off[e + 1])
        yield e, r, order[r] // plan.top_k if gather else torch.arange(off[e], off[e + 1], device=DEV)


def gated_ref(x, w, plan, gather, act, dh=None):
    """Values and bounds (without the results' own rounding) of h, dx, dw."""
    X, W, unit = x.detach().double(), w.detach().double(), UNIT[x.dtype]
    K, F, R = x.shape[1], w.shape[-1] // 2, x.shape[0] if plan is None else plan.num_rows
    h, bh = X.new_zeros(R, F), X.new_zeros(R, F)
    dx, bx, dw, bw = torch.zeros_like(X), torch.zeros_like(X), torch.zeros_like(W), torch.zeros_like(W)
    for e, r, rows in groups(plan, gather, x):
        a, we = X[rows], W[e]
        y, ey = a @ we, K * 2.0 ** -23 * (a.abs() @ we.abs())
        g, u, eg, eu = y[:, :F], y[:, F:], ey[:, :F], ey[:, F:]
        f, s = act_ref(act, g)
        ef = act_error(g) * f.abs() + 1.13 * eg + 1e-37
        # second derivatives are at most 1.2; relu's slope jumps where g is not known to be off zero
        es = act_error(g) * (s.abs() + f.abs()) + (1.2 * eg if act != "relu" else (g.abs() <= eg).double()) + 1e-37
        h[r], bh[r] = f * u, ef * u.abs() + f.abs() * eu + ef * eu
        if dh is None:
            continue
        d = dh[r].double()
        dy = torch.cat([d * u * s, d * f], 1)
        by = torch.cat([d.abs() * (es * (u.abs() + eu) + s.abs() * eu), d.abs() * ef], 1)
        by = by + 2 * unit * dy.abs() + 2 * TINY[x.dtype] * (1 + d.abs().repeat(1, 2))  # two roundings
        n = 2.0 ** -23
        dx.index_add_(0, rows, dy @ we.t())
        bx.index_add_(0, rows, (by + (2 * F + 32) * n * dy.abs()) @ we.abs().t())
        dw[e], bw[e] = a.t() @ dy, a.abs().t() @ (by + len(rows) * n * dy.abs())
    return h, bh, dx, bx, dw, bw


def close(got, ref, bound, dtype, norm=1.0):
    """norm: the roundings of a result, in the 2-norm over many values, beside its own."""
    assert got.dtype == dtype and got.shape == ref.shape
    err = (got.double() - ref).abs()
    over = err - (UNIT[dtype] * ref.abs() + bound + TINY[dtype])
    assert bool((over <= 0).all()), float(over.max())
    if ref.numel() > 500 and float(ref.norm()):
        assert float(err.norm()) <= (norm * UNIT[dtype] + 2.0 ** -18) * float(ref.norm())


def check(x, w, plan, gather, act, dh=None):
    if dh is not None:
        x.requires_grad_()
        w.requires_grad_()
    h = E.gated_matmul(x, w, plan, gather=gather, activation=act)
    rh, bh, rx, bx, rw, bw = gated_ref(x, w, plan, gather, act, dh)
    close(h.detach(), rh, bh, x.dtype)
    if plan is not None:
        assert not h[int(plan.offsets[-1]):].any()
    if dh is not None:
        dx, dw = torch.autograd.grad(h, (x, w), dh)
        close(dx, rx, bx, x.dtype, 3)
        close(dw, rw, bw, x.dtype, 3)
        with torch.no_grad():  # the form that keeps no slopes
            assert torch.equal(E.gated_matmul(x, w, plan, gather=gather, activation=act), h)
    E.check_device_errors()
    return h


@pytest.mark.parametrize("R", [1, 5, 33, 200, 700])
@pytest.mark.parametrize("K,F", [(64, 128), (8, 8), (200, 72), (37, 101), (520, 392), (1, 1), (1032, 300)])
@pytest.mark.parametrize("dtype", TYPES)
def test_dense(R, K, F, dtype):
    g = gen(R + K * F)
    x, w = randn(g, R, K, dtype=dtype), randn(g, K, 2 * F, dtype=dtype, scale=1.5 * K ** -0.5)
    check(x, w, None, False, ACTS[(R + K) % 4], randn(g, R, F, dtype=dtype))


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,F", [(64, 128), (200, 72), (37, 101), (520, 392)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(sizes, K, F, dtype, gather):
    s = SIZES[sizes]
    k = 2 if sum(s) % 2 == 0 else 1
    plan = make_plan(s, k, dropped=2 * k, seed=K)
    g = gen(K * F + len(s))
    x = randn(g, plan.num_tokens if gather else plan.num_rows, K, dtype=dtype)
    w = randn(g, len(s), K, 2 * F, dtype=dtype, scale=1.5 * K ** -0.5)
    check(x, w, plan, gather, ACTS[(len(s) + K + gather) % 4], randn(g, plan.num_rows, F, dtype=dtype))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations(act, dtype):
    """Every activation over its whole range, tails included: gate products from -60 to 60."""
    g = gen(len(act))
    R, F = 300, 64
    x = torch.zeros(R, 16, device=DEV)
    x[:, 0] = torch.linspace(-60, 60, R, device=DEV)
    x[:, 1] = 1.0
    w = torch.zeros(16, 2 * F, device=DEV)
    w[0, :F] = torch.linspace(0.03125, 1, F, device=DEV)
    w[1, F:] = randn(g, F)
    x, w = x.to(dtype), w.to(dtype)
    check(x, w, None, False, act, randn(g, R, F, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["transposed", "sliced", "padded", "offset", "odd", "broadcast"])
def test_layouts(dtype, layout):
    g = gen(3)
    n, K, F = 3, 72, 40
    plan = make_plan([30, 5, 111], 2)
    x = randn(g, plan.num_rows, K, dtype=dtype)
    w = randn(g, n, K, 2 * F, dtype=dtype, scale=K ** -0.5)
    if layout == "transposed":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "sliced":
        x = randn(g, plan.num_rows, 2 * K, dtype=dtype)[:, ::2]
        w = randn(g, n, K, 4 * F, dtype=dtype)[:, :, ::2]
    elif layout == "padded":
        x = randn(g, plan.num_rows, K + 8, dtype=dtype)[:, :K]
        w = randn(g, n, K, 2 * F + 24, dtype=dtype)[:, :, 8:8 + 2 * F]
    elif layout == "offset":
        x = randn(g, plan.num_rows * K + 1, dtype=dtype)[1:].view(plan.num_rows, K)
        w = randn(g, n * K * 2 * F + 1, dtype=dtype)[1:].view(n, K, 2 * F)
    elif layout == "odd":
        w = randn(g, n, K, 2 * F + 6, dtype=dtype)[:, :, 3:2 * F - 3]
        F -= 3
    else:
        w = randn(g, 1, K, 2 * F, dtype=dtype).expand(n, K, 2 * F)
    check(x.detach(), w.detach(), plan, False, "silu", randn(g, plan.num_rows, F, dtype=dtype))
    check(x.detach()[:90], w.detach()[1], None, False, "gelu", randn(g, 90, F, dtype=dtype))
    dh = randn(g, 90, F + 5, dtype=dtype)[:, 2:F + 2]
    check(x.detach()[:90], w.detach()[1], None, False, "gelu", dh)


def test_gradient_by_differences():
    g = gen(5)
    R, K, F = 6, 24, 20
    for act in ACTS[:3]:
        x, w = randn(g, R, K).requires_grad_(), randn(g, K, 2 * F, scale=K ** -0.5).requires_grad_()
        dh = randn(g, R, F)
        grads = torch.autograd.grad(E.gated_matmul(x, w, activation=act), (x, w), dh)

        def value(a, b):
            return (E.gated_matmul(a, b, activation=act).double() * dh.double()).sum()

        step = 2.0 ** -6
        for i in range(2):
            at = [x.detach(), w.detach()]
            way = randn(g, *at[i].shape)
            way = way / way.norm()
            up, dn = list(at), list(at)
            up[i], dn[i] = at[i] + step * way, at[i] - step * way
            rise = float(value(*up) - value(*dn)) / (2 * step)
            # h^2 / 6 of a third derivative (bounded by 8 a value here), 2^-20 of R F values of order 1 over the step
            assert abs(rise - float((grads[i].double() * way.double()).sum())) <= \
                step ** 2 / 6 * 8 * R * F ** 0.5 + 2.0 ** -20 * R * F / step


def test_empty():
    for R, K, F in ((0, 8, 8), (5, 0, 8), (5, 8, 0)):
        x = torch.zeros(R, K, device=DEV, requires_grad=True)
        w = torch.ones(K, 2 * F, device=DEV, requires_grad=True)
        h = E.gated_matmul(x, w)
        assert h.shape == (R, F) and not h.any()
        dx, dw = torch.autograd.grad(h, (x, w), torch.ones_like(h))
        assert dx.shape == x.shape and dw.shape == w.shape and not dw.any() and not dx.any()
    plan = make_plan([0, 0, 0], 1, dropped=4)
    for dtype in TYPES:
        x = torch.full((4, 16), math.nan, dtype=dtype, device=DEV, requires_grad=True)
        w = torch.ones(3, 16, 48, dtype=dtype, device=DEV, requires_grad=True)
        h = E.gated_matmul(x, w, plan)
        dx, dw = torch.autograd.grad(h, (x, w), torch.full_like(h, math.nan))
        assert not h.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_other_rows_stay_out(dtype):
    """Infinities and NaN of one expert's rows and weights, and of the rows of no expert, reach nothing else."""
    sizes = [20, 70, 300]
    plan = make_plan(sizes, 1, dropped=3)
    g = gen(7)
    x, w = randn(g, plan.num_rows, 40, dtype=dtype), randn(g, 3, 40, 48, dtype=dtype, scale=0.2)
    dh = randn(g, plan.num_rows, 24, dtype=dtype)
    x[25], x[393:], w[1, 3, 30], dh[30], dh[393:] = math.nan, math.nan, math.inf, math.inf, math.nan
    x.requires_grad_()
    w.requires_grad_()
    h = E.gated_matmul(x, w, plan)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    keep = torch.tensor([*range(20), *range(90, 390)], device=DEV)
    rh, bh, rx, bx, rw, bw = gated_ref(torch.nan_to_num(x.detach(), 0, 0, 0), torch.nan_to_num(w.detach(), 0, 0, 0),
                                       plan, False, "silu", torch.nan_to_num(dh, 0, 0, 0))
    close(h.detach()[keep], rh[keep], bh[keep], dtype)
    close(dx[keep], rx[keep], bx[keep], dtype, 3)
    close(dw[[0, 2]], rw[[0, 2]], bw[[0, 2]], dtype, 3)
    assert not h[390:].any() and not dx[390:].any()


def test_same_bits_streams_graph():
    plan = make_plan([40, 3, 900, 16, 0, 1], 2)
    g = gen(9)
    x = randn(g, plan.num_tokens, 512, dtype=torch.bfloat16).requires_grad_()
    w = randn(g, 6, 512, 528, dtype=torch.bfloat16, scale=0.05).requires_grad_()
    dh = randn(g, plan.num_rows, 264, dtype=torch.bfloat16)

    def step():
        h = E.gated_matmul(x, w, plan, gather=True)
        return (h.detach(), *torch.autograd.grad(h, (x, w), dh))

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    with torch.no_grad():
        x.mul_(-0.5)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))
    E.check_device_errors()


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(8, 12, device=DEV)
    plan = make_plan([3, 1], 1)
    for call in (lambda: E.gated_matmul(x, w[:7]), lambda: E.gated_matmul(x, w[:, :11]), lambda: E.gated_matmul(x[0], w),
                 lambda: E.gated_matmul(x, w[None]), lambda: E.gated_matmul(x, w, plan),
                 lambda: E.gated_matmul(x, w.expand(3, 8, 12), plan), lambda: E.gated_matmul(x, w, gather=True),
                 lambda: E.gated_matmul(x, w, activation="tanh"), lambda: E.gated_matmul(x, w.cpu()),
                 lambda: E.gated_matmul(x[:3], w.expand(2, 8, 12), plan)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: E.gated_matmul(x, w.half()), lambda: E.gated_matmul(x.double(), w.double()),
                 lambda: E.gated_matmul(x, w, 3)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(E.gated_matmul(x.requires_grad_(), w).sum(), x, create_graph=True)
        d.sum().backward()


CODE = {torch.float32: L.ES_F32, torch.bfloat16: L.ES_BF16, torch.float16: L.ES_F16}
LONG = [200, 701, 256, 0, 513, 390, 640, 511, 257]         # a mean past 112 rows
SHORT = [10 + 37 * i % 91 for i in range(58)] + [0, 129]   # 10 to 100 rows, none, and a tile and one
FEW = [i % 9 for i in range(80)] + [65]                    # up to 8 rows, and a tile and one


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("sizes,F,path", [(LONG, 2056, L.ES_GROUPED_WIDE), (LONG, 2049, L.ES_GROUPED_WIDE),
                                          (SHORT, 520, L.ES_GROUPED_MIDDLE), (SHORT, 517, L.ES_GROUPED_MIDDLE),
                                          (FEW, 520, L.ES_GROUPED_MIDDLE), (FEW, 517, L.ES_GROUPED_MIDDLE),
                                          (FEW, 100, L.ES_GROUPED_NARROW), (FEW, 97, L.ES_GROUPED_NARROW)])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_shapes(dtype, sizes, F, path, transposed, gather):
    """Every tile shape with ragged groups, several tiles a CTA, even and odd channels."""
    k = 2 if gather and sum(sizes) % 2 == 0 else 1
    plan = make_plan(sizes, k, dropped=4 * k)
    K = 136
    assert L.lib().es_gated_matmul_path(CODE[dtype], plan.num_experts, K, F, plan.num_rows) == path
    g = gen(F + len(sizes))
    x = randn(g, plan.num_tokens if gather else plan.num_rows, K, dtype=dtype)
    w = randn(g, len(sizes), *((2 * F, K) if transposed else (K, 2 * F)), dtype=dtype, scale=1.5 * K ** -0.5)
    w = w.transpose(1, 2) if transposed else w
    check(x, w, plan, gather, ACTS[(F + gather + 2 * transposed) % 4], randn(g, plan.num_rows, F, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("R,K,F", [(1, 2048, 512), (16, 4096, 130), (64, 1030, 257), (65, 520, 1024), (3, 16384, 40)])
@pytest.mark.parametrize("transposed", [False, True])
def test_split(dtype, R, K, F, transposed):
    """A decode step's few rows: a tile's depth shared by a cluster."""
    assert L.lib().es_gated_matmul_path(CODE[dtype], 0, K, F, R) == L.ES_GROUPED_SPLIT
    g = gen(R + F)
    x, w = randn(g, R, K, dtype=dtype), randn(g, K, 2 * F, dtype=dtype, scale=1.5 * K ** -0.5)
    if transposed:
        w = w.t().contiguous().t()
    check(x, w, None, False, ACTS[F % 4], randn(g, R, F, dtype=dtype))


@pytest.mark.parametrize("K", [16384, 16385])
def test_depth(K):
    """Up to one chain of sums the activation is in the product's kernel, deeper sums are made in fp32 first."""
    R, F = 300, 2000
    assert (L.lib().es_gated_matmul_path(L.ES_F16, 0, K, F, R) == L.ES_GATED_TWO) == (K > 16384)
    g = gen(K)
    x, w = randn(g, R, K, dtype=torch.float16), randn(g, K, 2 * F, dtype=torch.float16, scale=1.5 * K ** -0.5)
    check(x, w, None, False, "silu", None)
