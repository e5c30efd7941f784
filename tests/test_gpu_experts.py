"""Expert operators on the GPU against plain implementations in 64 bits.

Bounds, from the arithmetic and not from results: a value of type t is rounded
once (half a unit in the last place, ``UNIT``); a sum of n products in fp32 has
an error of at most ``n * 2**-23`` of the sum of the products' magnitudes (the
tensor cores may truncate, so a whole unit a step), and in the 2-norm over many
values far less.
"""

import math

import pytest
import torch

import einjax_b200 as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def near(got, ref, mag, n, dtype, extra=0.0):
    """got (dtype) against ref (64 bits), a sum of n products whose magnitudes add up to mag."""
    assert got.dtype == dtype and got.shape == ref.shape
    assert bool(torch.isfinite(got).all())
    err = (got.double() - ref).abs()
    bound = UNIT[dtype] * ref.abs() + (n * 2.0 ** -23 + extra) * mag + TINY[dtype]
    assert bool((err <= bound).all()), float((err - bound).max())
    norm = float(ref.norm())
    if norm:
        assert float(err.norm()) <= (UNIT[dtype] + 2.0 ** -19 + extra) * norm


# ------------------------------------------------------------------- routing

def route_ref(logits, k, renorm):
    x = logits.detach().double().cpu()
    T, n = x.shape
    experts = torch.full((T, k), -1, dtype=torch.int64)
    for t in range(T):
        row = [(-float(v), i) for i, v in enumerate(x[t].tolist()) if v > -math.inf]
        for j, (_, i) in enumerate(sorted(row)[:k]):
            experts[t, j] = i
    chosen = torch.zeros(T, n, dtype=torch.bool)
    for j in range(k):
        live = experts[:, j] >= 0
        chosen[torch.arange(T)[live], experts[live, j]] = True
    over = chosen if renorm else x > -math.inf
    p = torch.softmax(torch.where(over, x, -math.inf), 1).nan_to_num(0.0)
    w = torch.where(experts >= 0, p.gather(1, experts.clamp(min=0)), 0.0)
    return w, experts, p


@pytest.mark.parametrize("T,n,k", [(1, 1, 1), (1, 8, 8), (3, 33, 4), (130, 64, 8), (57, 128, 32), (9, 1000, 7),
                                   (5, 1024, 32), (4097, 60, 4)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renorm", [True, False])
def test_route(T, n, k, dtype, renorm):
    g = gen(T * n + k)
    x = randn(g, T, n, dtype=dtype, scale=2.0)
    x[torch.rand(T, n, generator=g, device=DEV) < 0.2] = -math.inf
    x[T // 2] = -math.inf  # a token with no expert at all
    x.requires_grad_()
    w, e = E.route_experts(x, k, renorm)
    rw, re, p = route_ref(x, k, renorm)
    assert w.dtype == torch.float32 and e.dtype == torch.int32
    assert torch.equal(e.cpu().long(), re)
    # exp and its argument (|l - m| < 32), at most 1024 terms summed 37 deep, a division
    tol = 2.0 ** -24 * (4 + 32 + 40 + 1)
    assert bool(((w.detach().cpu().double() - rw).abs() <= tol * rw + 1e-37).all())
    dw = torch.randn(T, k, generator=g, device=DEV)
    dx, = torch.autograd.grad(w, x, dw)
    full = torch.zeros(T, n, dtype=torch.float64)
    for j in range(k):
        live = re[:, j] >= 0
        full[torch.arange(T)[live], re[live, j]] = dw.cpu().double()[live, j]
    ref = p * (full - (p * full).sum(1, keepdim=True))
    mag = p * (full.abs() + (p * full.abs()).sum(1, keepdim=True))
    assert dx.dtype == dtype
    assert bool(((dx.cpu().double() - ref).abs() <= UNIT[dtype] * ref.abs() + 4 * tol * mag + TINY[dtype]).all())


@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_by_differences(renorm):
    g = gen(4)
    x = randn(g, 6, 20)
    dw = randn(g, 6, 3)
    x.requires_grad_()
    w, e = E.route_experts(x, 3, renorm)
    dx, = torch.autograd.grad(w, x, dw)
    h = 2.0 ** -7
    for i in range(20):
        step = torch.zeros_like(x)
        step[:, i] = h
        up, eu = E.route_experts(x.detach() + step, 3, renorm)
        dn, ed = E.route_experts(x.detach() - step, 3, renorm)
        same = (eu == e).all(1) & (ed == e).all(1)  # the choice itself is a step
        d = ((up - dn) * dw).sum(1) / (2 * h)
        # h^2 / 6 times a third derivative below 4 sum |dw|, and rounding over the step
        tol = (h * h + 2.0 ** -20 / h) * dw.abs().sum(1)
        assert bool(((d - dx[:, i]).abs() <= tol)[same].all())
    assert bool(same.any())


def test_route_special_values():
    lo = torch.finfo(torch.float32).min
    inf, nan = math.inf, math.nan
    x = torch.tensor([[1.0, 1.0, 1.0, 1.0],      # ties go to the lowest
                      [-0.0, 0.0, -0.0, -1.0],   # zeros are equal
                      [lo, lo, lo, lo],          # the lowest value is a logit
                      [-inf, lo, -inf, -inf],
                      [-inf, -inf, -inf, -inf],
                      [0.0, nan, 2.0, 1.0],
                      [0.0, inf, 2.0, 1.0],
                      [nan, nan, nan, nan]], device=DEV)
    for dtype in TYPES[:2]:
        y = x.to(dtype)
        y[(x == lo)] = torch.finfo(dtype).min
        w, e = E.route_experts(y, 2)
        assert e.cpu().tolist() == [[0, 1], [0, 1], [0, 1], [1, -1], [-1, -1], [2, 3], [1, 2], [-1, -1]]
        w = w.cpu()
        assert torch.equal(w[:5], torch.tensor([[0.5, 0.5], [0.5, 0.5], [0.5, 0.5], [1.0, 0.0], [0.0, 0.0]]))
        assert bool(w[5:].isnan().all())
        wa, ea = E.route_experts(y[:5], 2, renormalize=False)
        assert wa.cpu()[2].tolist() == [0.25, 0.25] and wa.cpu()[3].tolist() == [1.0, 0.0]


def test_route_strides_and_empty():
    g = gen(9)
    x = randn(g, 40, 96)
    for v in (x[::2], x[:, :50], x[:, ::3], x.t()):
        w, e = E.route_experts(v, 4)
        rw, re = E.route_experts(v.contiguous(), 4)
        assert torch.equal(e, re) and torch.equal(w, rw)
    w, e = E.route_experts(x[:0], 4)
    assert w.shape == e.shape == (0, 4)


# ----------------------------------------------------------------- row order

def layout_ref(experts, n):
    e = experts.cpu().long().reshape(-1)
    key = torch.where((e < 0) | (e >= n), n, e)
    order = torch.sort(key, stable=True).indices
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(key, minlength=n + 1)[:n].cumsum(0)])
    kept = torch.arange(e.numel()) < offsets[n]
    position = torch.empty_like(order)
    position[order] = torch.where(kept, torch.arange(e.numel()), -1)
    return offsets, torch.where(kept, order, -1), position.reshape(experts.shape)


@pytest.mark.parametrize("T,k,n", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (33, 3, 5), (512, 8, 60), (4096, 1, 128),
                                   (4097, 1, 128), (1024, 5, 1024), (40000, 8, 128), (100001, 2, 1000)])
@pytest.mark.parametrize("kind", ["even", "skewed", "none"])
def test_plan(T, k, n, kind):
    g = gen(T + n)
    e = torch.randint(0, n, (T, k), generator=g, device=DEV)
    if kind == "skewed":  # one expert has most of it, many have none, some choices are of no expert
        e = torch.where(torch.rand(T, k, generator=g, device=DEV) < 0.7, n // 2, e)
        e[torch.rand(T, k, generator=g, device=DEV) < 0.1] = -1
    elif kind == "none":
        e[:] = -1
    for dtype in (torch.int32, torch.int64):
        p = E.plan_experts(e.to(dtype), n)
        for got, want in zip((p.offsets, p.order, p.position), layout_ref(e, n)):
            assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)
    assert (p.num_experts, p.num_tokens, p.top_k, p.num_rows) == (n, T, k, T * k)
    assert torch.equal(p.counts.cpu(), (p.offsets[1:] - p.offsets[:-1]).cpu())
    E.check_device_errors()


@pytest.mark.parametrize("T", [10, 9000])
def test_plan_out_of_range(T):
    e = torch.zeros(T, 1, dtype=torch.int32, device=DEV)
    e[T // 2], e[3] = 7, -5
    p = E.plan_experts(e, 4)
    with pytest.raises(ValueError, match="es_expert_plan"):
        E.check_device_errors()
    E.check_device_errors()  # raised once
    for got, want in zip((p.offsets, p.order, p.position), layout_ref(e, 4)):
        assert torch.equal(got.cpu().long(), want)
    E.plan_experts(torch.tensor([[2 ** 32 + 1]], device=DEV), 4)
    with pytest.raises(ValueError):
        E.check_device_errors()


# ---------------------------------------------------------- grouped products

def make_plan(sizes, k=1, dropped=0, seed=0):
    """A plan whose experts have these rows; tokens are shuffled, k choices a token."""
    n = sum(sizes) + dropped
    assert n % k == 0
    g = torch.Generator().manual_seed(seed)
    e = torch.cat([torch.full((s,), i) for i, s in enumerate(sizes)] + [torch.full((dropped,), -1)]).int()
    e = e[torch.randperm(n, generator=g)].reshape(-1, k)
    return E.plan_experts(e.to(DEV), len(sizes))


def grouped_ref(x, w, plan, gather, dy=None):
    """(y, |y|, dx, |dx|, dw, |dw|) in 64 bits; |.|: of the operands' magnitudes."""
    off, order = plan.offsets.tolist(), plan.order.long()
    X, W = x.detach().double(), w.detach().double()
    y, my = (X.new_zeros(plan.num_rows, w.shape[2]) for _ in range(2))
    G = dy.double() if dy is not None else y
    dx, mx, dw, mw = torch.zeros_like(X), torch.zeros_like(X), torch.zeros_like(W), torch.zeros_like(W)
    for e in range(plan.num_experts):
        r = slice(off[e], off[e + 1])
        rows = order[r] // plan.top_k if gather else torch.arange(off[e], off[e + 1], device=DEV)
        a = X[rows]
        y[r], my[r] = a @ W[e], a.abs() @ W[e].abs()
        dx.index_add_(0, rows, G[r] @ W[e].t())
        mx.index_add_(0, rows, G[r].abs() @ W[e].abs().t())
        dw[e], mw[e] = a.t() @ G[r], a.abs().t() @ G[r].abs()
    return y, my, dx, mx, dw, mw


SIZES = {
    "one": [1],
    "ones": [1, 0, 1, 1, 0, 1],
    "few": [3, 0, 17, 40, 0, 0, 8, 20],
    "edges": [16, 31, 32, 33, 64, 65, 127, 1],
    "big": [300, 1, 0, 511, 129, 257, 0, 2],
    "last": [0, 0, 0, 260],
    "uneven": [30, 0, 0, 0, 1, 2, 0, 9],
}


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N", [(64, 128), (8, 8), (200, 72), (37, 101), (520, 392), (1, 1)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(sizes, K, N, dtype, gather):
    s = SIZES[sizes]
    k = 2 if sum(s) % 2 == 0 else 1
    plan = make_plan(s, k, dropped=2 * k, seed=K)
    g = gen(K * N + len(s))
    x = randn(g, plan.num_tokens if gather else plan.num_rows, K, dtype=dtype).requires_grad_()
    w = randn(g, len(s), K, N, dtype=dtype, scale=K ** -0.5).requires_grad_()
    dy = randn(g, plan.num_rows, N, dtype=dtype)
    y = E.grouped_matmul(x, w, plan, gather=gather)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, my, rx, mx, rw, mw = grouped_ref(x, w, plan, gather, dy)
    near(y.detach(), ry, my, K, dtype)
    near(dx, rx, mx, N + k, dtype)
    near(dw, rw, mw, max(s), dtype)
    kept = sum(s)
    assert not y[kept:].any()
    E.check_device_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [1, 4, 0, 5, 8, 9], [0, 0, 25, 0, 0, 0]])
@pytest.mark.parametrize("K,N", [(2100, 132), (1028, 1000), (1024, 64), (4, 4), (2052, 20)])
def test_grouped_few_rows(dtype, sizes, K, N):
    """Groups of a few rows, depths past a chunk, both orders of the weights."""
    plan = make_plan(sizes, 1, dropped=2)
    g = gen(K + N)
    x = randn(g, plan.num_tokens, K, dtype=dtype).requires_grad_()
    w = randn(g, len(sizes), K, N, dtype=dtype, scale=K ** -0.5)
    dy = randn(g, plan.num_rows, N, dtype=dtype)
    for v in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        v = v.detach().requires_grad_()
        y = E.grouped_matmul(x, v, plan, gather=True)
        dx, dw = torch.autograd.grad(y, (x, v), dy)
        ry, my, rx, mx, rw, mw = grouped_ref(x, v, plan, True, dy)
        near(y.detach(), ry, my, K, dtype)
        near(dx, rx, mx, N + 1, dtype)
        near(dw, rw, mw, max(sizes), dtype)
        assert not y[sum(sizes):].any()


@pytest.mark.parametrize("experts,rows", [(40, 300), (7, 41), (64, 9)])
def test_grouped_few_rows_of_one_expert(experts, rows):
    """All rows at one expert (more than its share of the launch) or all but one."""
    g = gen(rows)
    K, N = 1032, 76
    for other in (0, 1):
        sizes = [0] * experts
        sizes[experts // 2], sizes[-1] = rows - other, other
        plan = make_plan(sizes, 1, dropped=1)
        x = randn(g, plan.num_tokens, K, dtype=torch.float32).requires_grad_()
        w = randn(g, experts, K, N, dtype=torch.float32, scale=K ** -0.5).requires_grad_()
        dy = randn(g, plan.num_rows, N, dtype=torch.float32)
        y = E.grouped_matmul(x, w, plan, gather=True)
        dx, = torch.autograd.grad(y, x, dy)
        ry, my, rx, mx, _, _ = grouped_ref(x, w, plan, True, dy)
        near(y.detach(), ry, my, K, torch.float32)
        near(dx, rx, mx, N + 1, torch.float32)
        assert not y[rows:].any()


@pytest.mark.parametrize("K,N", [(388, 72), (768, 200), (20, 4), (1500, 64)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_grouped_few_rows_strides(K, N, pad):
    """Several tiles of rows an expert, x and weights as views: offset, with a longer pitch, one of them not 16 bytes."""
    sizes = [16, 17, 0, 31, 33, 2, 8]
    plan = make_plan(sizes, 1, dropped=3)
    g = gen(K + pad)
    base = randn(g, plan.num_tokens, K + 2 * pad, dtype=torch.float32)
    x = base[:, pad:pad + K].detach().requires_grad_()
    wbase = randn(g, len(sizes), K + 4, N + 8, dtype=torch.float32, scale=K ** -0.5)
    w = wbase[:, 4:, 4:4 + N].detach().requires_grad_()
    dy = randn(g, plan.num_rows, N, dtype=torch.float32)
    for gather in (True, False):
        y = E.grouped_matmul(x, w, plan, gather=gather)
        dx, = torch.autograd.grad(y, x, dy)
        ry, my, rx, mx, _, _ = grouped_ref(x, w, plan, gather, dy)
        near(y.detach(), ry, my, K, torch.float32)
        near(dx, rx, mx, N + 1, torch.float32)
        assert not y[sum(sizes):].any()


def test_grouped_few_rows_largest():
    """Values next to the type's largest, whose first plane would be an infinity."""
    big = torch.finfo(torch.float32).max
    plan = make_plan([2, 1], 1)
    g = gen(5)
    x = randn(g, 3, 64, dtype=torch.float32) * 2.0 ** -10
    w = randn(g, 2, 64, 8, dtype=torch.float32)
    w[0, 3, 2], w[1, 63, 7] = big, -big
    y = E.grouped_matmul(x, w, plan)
    ry, my = grouped_ref(x, w, plan, False, torch.zeros(3, 8, device=DEV))[:2]
    near(y, ry, my, 64, torch.float32)


@pytest.mark.parametrize("K,N", [(2100, 132), (1028, 20), (12, 64)])
def test_grouped_few_rows_infinite(K, N):
    """An infinity at the end of a row's depth makes infinities, and leaves the other rows alone."""
    plan = make_plan([3, 0, 2], 1)
    g = gen(K)
    x = randn(g, 5, K, dtype=torch.float32)
    w = randn(g, 3, K, N, dtype=torch.float32).abs() + 1
    bad = x.clone()
    bad[1, K - 1], bad[4, 0] = math.inf, -math.inf
    for v in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        y, want = E.grouped_matmul(bad, v, plan), E.grouped_matmul(x, v, plan)
        assert bool((y[1] == math.inf).all()) and bool((y[4] == -math.inf).all())
        assert torch.equal(y[[0, 2, 3]], want[[0, 2, 3]])


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_many_experts(dtype):
    """As many experts as there may be, most of them without rows."""
    sizes = [0] * 1024
    sizes[3], sizes[500], sizes[501], sizes[1023] = 5, 40, 1, 18
    plan = make_plan(sizes, 2)
    g = gen(14)
    x = randn(g, plan.num_tokens, 40, dtype=dtype).requires_grad_()
    w = randn(g, 1024, 40, 24, dtype=dtype).requires_grad_()
    dy = randn(g, plan.num_rows, 24, dtype=dtype)
    y = E.grouped_matmul(x, w, plan, gather=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, my, rx, mx, rw, mw = grouped_ref(x, w, plan, True, dy)
    near(y.detach(), ry, my, 40, dtype)
    near(dx, rx, mx, 24 + 2, dtype)
    near(dw, rw, mw, 40, dtype)
    wq, ws = E.quantize_experts(w)
    q, s = E.quantize_rows(x)
    check_int8(E.int8_matmul(q, s, wq, ws, plan, gather=True, out_dtype=dtype),
               int8_ref(q, s, wq, ws, plan, True), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_long(dtype):
    """Depths where a sum's own rounding shows, and more tiles than SMs."""
    plan = make_plan([700, 33, 0, 1400, 5, 301], 1, dropped=3)
    g = gen(3)
    K, N = 2048, 1160
    x = randn(g, plan.num_rows, K, dtype=dtype).requires_grad_()
    w = randn(g, 6, K, N, dtype=dtype, scale=K ** -0.5).requires_grad_()
    dy = randn(g, plan.num_rows, N, dtype=dtype)
    y = E.grouped_matmul(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, my, rx, mx, rw, mw = grouped_ref(x, w, plan, False, dy)
    near(y.detach(), ry, my, K, dtype)
    near(dx, rx, mx, N, dtype)
    near(dw, rw, mw, 1400, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["transposed", "sliced", "padded", "strided", "offset", "broadcast", "permuted",
                                    "turned"])
def test_grouped_layouts(dtype, layout):
    """Weights and rows that lie otherwise in memory give what their copies give."""
    plan = make_plan([5, 130, 0, 64], 1)
    g = gen(11)
    K, N, n = 96, 136, plan.num_rows
    x = randn(g, n, K, dtype=dtype)
    w = randn(g, 4, K, N, dtype=dtype, scale=K ** -0.5)
    if layout == "transposed":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "sliced":  # part of a wider matrix
        w = randn(g, 4, K, 2 * N, dtype=dtype, scale=K ** -0.5)[:, :, N:]
    elif layout == "padded":  # rows of x further apart
        x = randn(g, n, K + 24, dtype=dtype)[:, :K]
    elif layout == "strided":
        w, x = randn(g, 4, K, 2 * N, dtype=dtype)[:, :, ::2], randn(g, n, 2 * K, dtype=dtype)[:, ::2]
    elif layout == "offset":  # a base address that no 16-byte load may start at
        w = randn(g, 4 * K * N + 1, dtype=dtype)[1:].reshape(4, K, N)
        x = randn(g, n * K + 1, dtype=dtype)[1:].reshape(n, K)
    elif layout == "permuted":  # the experts' matrices interleaved row by row
        w = randn(g, K, 4, N, dtype=dtype, scale=K ** -0.5).transpose(0, 1)
    elif layout == "turned":  # the experts innermost
        w = randn(g, K, N, 4, dtype=dtype, scale=K ** -0.5).permute(2, 0, 1)
    else:
        w, x = w[:1].expand(4, K, N), x[:1].expand(n, K)
    x.requires_grad_()
    w.requires_grad_()
    dy = randn(g, N, n, dtype=dtype).t()
    y = E.grouped_matmul(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, my, rx, mx, rw, mw = grouped_ref(x, w, plan, False, dy)
    near(y.detach(), ry, my, K, dtype)
    near(dx, rx, mx, N, dtype)
    near(dw, rw, mw, 130, dtype)
    if layout == "transposed":
        assert dw.stride() == w.stride()


def test_grouped_broadcast_leaf():
    """The gradient of a matrix that all experts share is the sum over them."""
    plan = make_plan([5, 13, 0, 30], 2)
    g = gen(12)
    w = randn(g, 32, 48).requires_grad_()
    x = randn(g, plan.num_tokens, 32).requires_grad_()
    y = E.grouped_matmul(x, w.expand(4, 32, 48), plan, gather=True)
    dy = randn(g, *y.shape)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    _, _, rx, mx, rw, mw = grouped_ref(x, w.expand(4, 32, 48), plan, True, dy)
    near(dx, rx, mx, 50, torch.float32)
    near(dw, rw.sum(0), mw.sum(0), 34, torch.float32)


def test_grouped_gradient_by_differences():
    """The product is bilinear: a difference of two calls is the gradient up to rounding."""
    plan = make_plan([3, 0, 9, 4], 2)
    g = gen(13)
    x, w = randn(g, plan.num_tokens, 24).requires_grad_(), randn(g, 4, 24, 20).requires_grad_()
    dy = randn(g, plan.num_rows, 20)
    dx, dw = torch.autograd.grad(E.grouped_matmul(x, w, plan, gather=True), (x, w), dy)
    ux, uw = randn(g, *x.shape), randn(g, *w.shape)

    def f(a, b):
        return float((E.grouped_matmul(x.detach() + a * ux, w.detach() + b * uw, plan, gather=True).double()
                      * dy.double()).sum())

    scale = float(dy.abs().sum()) * 24 * 4
    assert abs((f(1, 0) - f(-1, 0)) / 2 - float((dx * ux).sum())) <= 2.0 ** -18 * scale
    assert abs((f(0, 1) - f(0, -1)) / 2 - float((dw * uw).sum())) <= 2.0 ** -18 * scale


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_empty(dtype):
    for sizes, dropped, K, N in ([0, 0], 0, 16, 16), ([0, 0], 70, 16, 16), ([3, 4], 0, 0, 16), ([3, 4], 0, 16, 0):
        plan = make_plan(sizes, 1, dropped)
        x = torch.ones(plan.num_rows, K, dtype=dtype, device=DEV, requires_grad=True)
        w = torch.ones(2, K, N, dtype=dtype, device=DEV, requires_grad=True)
        y = E.grouped_matmul(x, w, plan)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert y.shape == (plan.num_rows, N)
        if K == 0 or N == 0 or not sum(sizes):
            assert not y.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_other_rows_stay_out(dtype):
    """Infinities and NaN in one expert's rows or weights reach no other expert, and no empty row."""
    sizes = [5, 70, 3, 0, 40]
    plan = make_plan(sizes, 1, dropped=4)
    g = gen(17)
    K, N = 72, 136
    x, w = randn(g, plan.num_rows, K, dtype=dtype), randn(g, 5, K, N, dtype=dtype)
    dy = randn(g, plan.num_rows, N, dtype=dtype)
    off = plan.offsets.tolist()
    clean = [t.clone().requires_grad_() for t in (x, w)]
    want = E.grouped_matmul(*clean, plan)
    wdx, wdw = torch.autograd.grad(want, clean, dy)
    for bad in (math.nan, math.inf):
        xb, wb, db = x.clone(), w.clone(), dy.clone()
        xb[off[1]:off[2]], wb[1], wb[3], db[off[1]:off[2]] = bad, bad, bad, bad
        xb[off[5]:], db[off[5]:] = bad, bad
        xb.requires_grad_()
        wb.requires_grad_()
        y = E.grouped_matmul(xb, wb, plan)
        dx, dw = torch.autograd.grad(y, (xb, wb), db)
        keep = torch.ones(plan.num_rows, dtype=torch.bool, device=DEV)
        keep[off[1]:off[2]] = False
        assert torch.equal(y[keep], want[keep]) and torch.equal(dx[keep], wdx[keep])
        assert not bool(torch.isfinite(y[~keep]).any())
        for e in (0, 2, 3, 4):
            assert torch.equal(dw[e], wdw[e])


def test_grouped_bounds_offsets():
    """Offsets and orders that point outside are bounded: rows inside are right, nothing faults."""
    plan = make_plan([4, 4], 1)
    x, w = torch.ones(8, 16, device=DEV), torch.ones(2, 16, 8, device=DEV)
    off = torch.tensor([-5, 4, 1000], dtype=torch.int32, device=DEV)
    y = E.grouped_matmul(x, w, E.ExpertPlan(off, plan.order, plan.position))
    assert bool((y == 16).all())
    order = plan.order.clone()
    order[2] = 10 ** 6
    y = E.grouped_matmul(x, w, E.ExpertPlan(plan.offsets, order, plan.position), gather=True)
    assert not y[2].any() and bool((y[3:] == 16).all())
    torch.cuda.synchronize()


def test_grouped_refusals():
    plan = make_plan([3, 5], 2)
    x, w = torch.ones(4, 16, device=DEV), torch.ones(2, 16, 8, device=DEV)
    E.grouped_matmul(x, w, plan, gather=True)
    for bad, args in ((ValueError, (x, w, plan)), (ValueError, (x[:, :8], w, plan, True)),
                      (ValueError, (x, w[:1], plan, True)), (ValueError, (x, w[0], plan, True)),
                      (TypeError, (x.double(), w.double(), plan, True)), (TypeError, (x.half(), w, plan, True)),
                      (TypeError, (x, w, plan.offsets, True)), (ValueError, (x.cpu(), w, plan, True)),
                      (TypeError, (x.tolist(), w, plan, True))):
        with pytest.raises(bad):
            E.grouped_matmul(*args)


# ------------------------------------------------------ weighted sum to tokens

@pytest.mark.parametrize("T,k,D", [(1, 1, 1), (1, 8, 4096), (7, 3, 37), (130, 2, 264), (33, 12, 1000), (5, 32, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_combine(T, k, D, dtype):
    g = gen(T + D)
    e = torch.randint(-1, 6, (T, k), generator=g, device=DEV).int()
    plan = E.plan_experts(e, 6)
    y = randn(g, T * k, D, dtype=dtype).requires_grad_()
    w = torch.rand(T, k, generator=g, device=DEV).requires_grad_()
    out = E.combine_experts(y, w, plan)
    dout = randn(g, T, D, dtype=dtype)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    at = plan.position.long()
    Y = torch.where(at[..., None] >= 0, y.detach().double()[at.clamp(min=0)], 0.0)
    W, G = w.detach().double(), dout.double()
    near(out.detach(), (Y * W[..., None]).sum(1), (Y.abs() * W[..., None]).sum(1), k, dtype)
    near(dw, (Y * G[:, None]).sum(2), (Y * G[:, None]).abs().sum(2), D, torch.float32)
    ref = torch.zeros(T * k, D, dtype=torch.float64, device=DEV)
    ref[at[at >= 0]] = (W[..., None] * G[:, None])[at >= 0]
    near(dy, ref, ref.abs(), 1, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_combine_layouts(dtype):
    plan = make_plan([9, 0, 11, 20], 4)
    g = gen(5)
    w = torch.rand(10, 4, generator=g, device=DEV)
    wide = randn(g, 40, 96, dtype=dtype)
    odd = randn(g, 40 * 64 + 1, dtype=dtype)
    for y in (wide[:, :64], wide[:, 1:65], wide[:, ::2], odd[1:].reshape(40, 64), wide[:1].expand(40, 96)):
        for dout in (randn(g, 10, y.shape[1], dtype=dtype), randn(g, y.shape[1], 10, dtype=dtype).t(),
                     randn(g, 1, y.shape[1], dtype=dtype).expand(10, -1)):
            a, b = y.detach().requires_grad_(), y.detach().contiguous().clone().requires_grad_()
            wa, wb = w.clone().requires_grad_(), w.clone().t().contiguous().t().requires_grad_()
            oa, ob = E.combine_experts(a, wa, plan), E.combine_experts(b, wb, plan)
            assert torch.equal(oa, ob)
            for p, q in zip(torch.autograd.grad(oa, (a, wa), dout),
                            torch.autograd.grad(ob, (b, wb), dout.contiguous().clone())):
                # the same sums, in pieces of 16 bytes or of one value
                assert bool(((p.double() - q.double()).abs() <= 96 * 2.0 ** -22 * 16).all())


def test_combine_past_32_bits():
    """Rows whose element offsets pass 2^31."""
    rows, D = 550_000, 4096
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    y = torch.empty(rows, D, dtype=torch.bfloat16, device=DEV)
    y[-3:] = torch.arange(3, device=DEV)[:, None] + 1
    position = torch.full((rows, 1), -1, dtype=torch.int32, device=DEV)
    position[0], position[rows - 1] = rows - 1, rows - 3
    plan = E.ExpertPlan(torch.tensor([0, rows], dtype=torch.int32, device=DEV),
                        torch.zeros(rows, dtype=torch.int32, device=DEV), position)
    out = E.combine_experts(y, torch.full((rows, 1), 2.0, device=DEV), plan)
    assert bool((out[0] == 6).all()) and bool((out[rows - 1] == 2).all()) and not out[1:rows - 1].any()
    # the product's gathered rows: a group at the end of a long x
    w = torch.ones(1, D, 16, dtype=torch.bfloat16, device=DEV)
    p2 = E.ExpertPlan(torch.tensor([0, 2], dtype=torch.int32, device=DEV),
                      torch.tensor([rows - 1, rows - 2], dtype=torch.int32, device=DEV).repeat(rows // 2),
                      torch.zeros(rows, 1, dtype=torch.int32, device=DEV))
    got = E.grouped_matmul(y, w, p2, gather=True)
    assert bool((got[0] == 3 * D).all()) and bool((got[1] == 2 * D).all())


def test_combine_refusals():
    plan = make_plan([3, 5], 2)
    y, w = torch.ones(8, 16, device=DEV), torch.ones(4, 2, device=DEV)
    E.combine_experts(y, w, plan)
    for bad, args in ((ValueError, (y[:7], w, plan)), (ValueError, (y, w[:, :1], plan)),
                      (TypeError, (y, w.half(), plan)), (TypeError, (y.long(), w, plan)), (TypeError, (y, w, None)),
                      (ValueError, (y, w.cpu(), plan))):
        with pytest.raises(bad):
            E.combine_experts(*args)


# ------------------------------------------------------------ 8-bit products

def quant_ref(x):
    x = x.double()
    s = (x.abs().amax(1) / 127).float() if x.shape[1] else torch.zeros(x.shape[0], device=DEV)
    q = torch.where(s[:, None] > 0, torch.round((x.float() / s[:, None])), 0.0)
    return q.clamp(-127, 127).to(torch.int8), s


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 8), (17, 129), (64, 4096), (5, 9000), (2, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize(rows, width, dtype):
    g = gen(rows + width)
    x = randn(g, rows, width, dtype=dtype, scale=3.0)
    if rows > 2:
        x[1] = 0
    for v in (x, randn(g, rows, width + 16, dtype=dtype)[:, 8:8 + width], randn(g, width, rows, dtype=dtype).t()):
        q, s = E.quantize_rows(v)
        rq, rs = quant_ref(v)
        assert q.dtype == torch.int8 and s.dtype == torch.float32
        assert torch.equal(s, rs) and torch.equal(q, rq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_every_value(dtype):
    """Every finite value of a type under largest values of every kind of mantissa, and next to the type's ends."""
    every = torch.arange(2 ** 15, dtype=torch.int32, device=DEV).to(torch.int16).view(dtype)
    every = every[every.isfinite()]
    n = 128 if dtype == torch.bfloat16 else 1024
    peaks = [(1 + m / n) * 2.0 ** e for e in (-3, 0, 9) for m in range(0, n, 1 if n == 128 else 7)]
    peaks += every[[1, 2, 3, 77, 300, -300, -2, -1]].tolist()
    for some in torch.tensor(peaks, dtype=torch.float64).split(32):
        top = some.to(DEV, dtype)
        x = torch.where(every[None, :] <= top[:, None], every[None, :], top[:, None])
        x[:, ::2] = -x[:, ::2]
        q, s = E.quantize_rows(x)
        rq, rs = quant_ref(x)
        assert torch.equal(s, rs) and torch.equal(q, rq)


def test_quantize_special():
    x = torch.tensor([[1.0, math.inf, 0], [math.nan, 1.0, 2.0], [0, 0, 0], [2.0 ** -149, 0, 0], [-3.0, 1.5, 3.0]],
                     device=DEV)
    q, s = E.quantize_rows(x)
    assert bool(s[:2].isnan().all()) and not q[:2].any()
    assert s[2] == 0 and not q[2].any() and not q[3].any()  # the smallest value's scale is below the type
    assert q[4].tolist() == [-127, 64, 127]
    y = E.int8_matmul(q, s, torch.ones(4, 3, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV),
                      out_dtype=torch.float32)
    assert bool(y[:2].isnan().all()) and not y[2:4].any()


def int8_ref(q, s, wq, ws, plan, gather):
    if plan is None:
        return (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()
    off, order = plan.offsets.tolist(), plan.order.long()
    y = torch.zeros(plan.num_rows, wq.shape[1], dtype=torch.float64, device=DEV)
    for e in range(plan.num_experts):
        r = slice(off[e], off[e + 1])
        rows = order[r] // plan.top_k if gather else torch.arange(off[e], off[e + 1], device=DEV)
        y[r] = (q[rows].double() @ wq[e].double().t()) * s[rows].double()[:, None] * ws[e].double()
    return y


def check_int8(y, ref, dtype):
    # the sum to fp32, two products and the last rounding
    assert y.dtype == dtype
    err = (y.double() - ref).abs()
    assert bool((err <= (UNIT[dtype] + 3 * 2.0 ** -24) * ref.abs() + TINY[dtype]).all())


def int8s(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


@pytest.mark.parametrize("rows", [1, 3, 33, 200, 700])
@pytest.mark.parametrize("K,N", [(16, 8), (128, 128), (1040, 264), (100, 37), (4096, 1000), (5, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_dense(rows, K, N, dtype):
    g = gen(rows + K + N)
    q, wq = int8s(g, rows, K), int8s(g, N, K)
    q[0], wq[0] = 127, -127  # the largest sum
    s, ws = torch.rand(rows, generator=g, device=DEV) * 2.0 ** -10, torch.rand(N, generator=g, device=DEV) * 2.0 ** -8
    y = E.int8_matmul(q, s, wq, ws, out_dtype=dtype)
    check_int8(y, int8_ref(q, s, wq, ws, None, False), dtype)


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N", [(64, 128), (16, 8), (208, 72), (37, 101)])
@pytest.mark.parametrize("gather", [False, True])
def test_int8_grouped(sizes, K, N, gather):
    n = SIZES[sizes]
    k = 2 if sum(n) % 2 == 0 else 1
    plan = make_plan(n, k, dropped=2 * k)
    g = gen(K + len(n))
    q, wq = int8s(g, plan.num_tokens if gather else plan.num_rows, K), int8s(g, len(n), N, K)
    s, ws = torch.rand(q.shape[0], generator=g, device=DEV), torch.rand(len(n), N, generator=g, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        y = E.int8_matmul(q, s * 2.0 ** -12, wq, ws, plan, gather=gather, out_dtype=dtype)
        check_int8(y, int8_ref(q, s * 2.0 ** -12, wq, ws, plan, gather), dtype)
    E.check_device_errors()


def test_int8_deepest():
    """The largest sums that 32-bit integers hold, and one step more, which is refused."""
    K = 131071
    for depth in (K, K - 15):  # odd rows are laid out anew, the others read as they lie
        q = torch.full((3, depth), -128, dtype=torch.int8, device=DEV)
        wq = torch.full((17, depth), -128, dtype=torch.int8, device=DEV)
        q[1], wq[5] = 127, 127
        one = torch.ones(17, device=DEV)
        y = E.int8_matmul(q, one[:3], wq, one, out_dtype=torch.float32)
        check_int8(y, int8_ref(q, one[:3], wq, one, None, False), torch.float32)
    q = torch.zeros(1, K + 1, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError):
        E.int8_matmul(q, torch.ones(1, device=DEV), q, torch.ones(1, device=DEV))


def test_int8_layouts():
    g = gen(2)
    q, wq = int8s(g, 50, 192), int8s(g, 40, 192)
    s, ws = torch.rand(50, generator=g, device=DEV), torch.rand(40, generator=g, device=DEV)
    for a, b in ((q[:, 32:160], wq[:, 32:160]), (q[:, 1:129], wq[:, 1:129]), (q[:, ::2], wq[:, ::2]),
                 (q[::2], wq), (q[:1].expand(50, 192), wq[:1].expand(40, 192))):
        sa = s[::2] if a.shape[0] == 25 else s
        y = E.int8_matmul(a, sa, b, ws, out_dtype=torch.float32)
        check_int8(y, int8_ref(a, sa, b, ws, None, False), torch.float32)


def test_int8_refusals():
    g = gen(1)
    q, wq, s, ws = int8s(g, 4, 16), int8s(g, 8, 16), torch.ones(4, device=DEV), torch.ones(8, device=DEV)
    E.int8_matmul(q, s, wq, ws)
    for bad, args, kw in ((TypeError, (q.int(), s, wq, ws), {}), (TypeError, (q, s.half(), wq, ws), {}),
                          (ValueError, (q, s, wq[:, :8], ws), {}), (ValueError, (q, s[:2], wq, ws), {}),
                          (ValueError, (q, s, wq, ws[:2]), {}), (ValueError, (q, s, wq, ws), {"gather": True}),
                          (TypeError, (q, s, wq, ws), {"out_dtype": torch.float64}),
                          (ValueError, (q, s, wq, ws, make_plan([2, 2])), {}),
                          (ValueError, (torch.zeros(1, 133153, dtype=torch.int8, device=DEV), s[:1],
                                        torch.zeros(8, 133153, dtype=torch.int8, device=DEV), ws), {})):
        with pytest.raises(bad):
            E.int8_matmul(*args, **kw)


def test_route_and_plan_refusals():
    x = torch.ones(4, 16, device=DEV)
    for bad, args in ((ValueError, (x, 0)), (ValueError, (x, 17)), (ValueError, (x[0], 2)), (TypeError, (x.int(), 2)),
                      (ValueError, (x.cpu(), 2)), (ValueError, (torch.ones(1, 1025, device=DEV), 2)),
                      (ValueError, (torch.ones(1, 64, device=DEV), 33))):
        with pytest.raises(bad):
            E.route_experts(*args)
    e = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    for bad, args in ((ValueError, (e, 0)), (ValueError, (e, 1025)), (ValueError, (e[0], 4)),
                      (TypeError, (e.float(), 4))):
        with pytest.raises(bad):
            E.plan_experts(*args)
    with pytest.raises(ValueError):
        E.ExpertPlan(e.reshape(-1), e.reshape(-1), e[:2])
    with pytest.raises(TypeError):
        E.ExpertPlan(e.reshape(-1).long(), e.reshape(-1), e)


# ---------------------------------------------------------------- all together

def mlp_ref(x, router, w_in, w_out, experts, weights):
    out = x.new_zeros(x.shape[0], w_out.shape[2])
    for j in range(experts.shape[1]):
        for e in range(router.shape[1]):
            rows = (experts[:, j] == e).nonzero()[:, 0]
            h = x[rows] @ w_in[e]
            f = h.shape[1] // 2
            out = out.index_add(0, rows, (torch.nn.functional.silu(h[:, :f]) * h[:, f:]) @ w_out[e]
                                * weights[rows, j, None])
    return out


def test_expert_mlp():
    """Forward and every gradient of the layer against autograd in 64 bits; the 8-bit form within its rounding."""
    g = gen(6)
    T, D, F, n, k = 150, 64, 96, 6, 2
    x, router = randn(g, T, D).requires_grad_(), randn(g, D, n, scale=D ** -0.5).requires_grad_()
    w_in = randn(g, n, D, 2 * F, scale=D ** -0.5).requires_grad_()
    w_out = randn(g, n, F, D, scale=F ** -0.5).requires_grad_()
    out = E.expert_mlp(x, router, w_in, w_out, k)
    dout = randn(g, T, D)
    got = torch.autograd.grad(out, (x, router, w_in, w_out), dout)
    ref_in = [t.detach().double().requires_grad_() for t in (x, router, w_in, w_out)]
    logits = ref_in[0] @ ref_in[1]
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    ref = mlp_ref(*ref_in, top.indices[:, :k], torch.softmax(top.values[:, :k], 1))
    want = torch.autograd.grad(ref, ref_in, dout.double())
    for a, b in zip((out.detach(), *got), (ref.detach(), *want)):
        # a chain of five operators, each within 2^-19 in the norm, whose factors are of order one
        assert float((a.double() - b).norm()) <= 2.0 ** -15 * float(b.norm())
    q = E.expert_mlp(x.detach(), router.detach(), E.quantize_experts(w_in), E.quantize_experts(w_out), k)
    # four operands in 8 bits: half a step of max / 127, the maximum about 3 deviations: 0.7% each
    assert float((q.double() - ref.detach()).norm()) <= 0.03 * float(ref.detach().norm())


def test_example_trains_and_serves():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_mlp.py")
    spec = importlib.util.spec_from_file_location("expert_mlp_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(steps=60, tokens=300)
    assert got["last"] < 0.7 * got["first"]
    # as in test_expert_mlp: four operands in 8 bits, half a step of max / 127 each, and bf16 beside it
    assert got["int8_off"] < 0.03


def test_streams_and_graph():
    """Calls on another stream, and captured in a CUDA graph, give what they give on the default stream."""
    plan = make_plan([40, 0, 200, 16], 2)
    g = gen(8)
    x = randn(g, plan.num_tokens, 128, dtype=torch.bfloat16)
    w = randn(g, 4, 128, 136, dtype=torch.bfloat16)
    weights = torch.rand(plan.num_tokens, 2, generator=g, device=DEV)
    logits = randn(g, plan.num_tokens, 4)

    def step():
        wt, ex = E.route_experts(logits, 2)
        p = E.plan_experts(ex, 4)
        return (E.combine_experts(E.grouped_matmul(x, w, p, gather=True), wt, p),
                E.combine_experts(E.grouped_matmul(x, w, plan, gather=True), weights, plan))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, held):
        assert torch.equal(a, b) and torch.equal(a, c)
    del graph


def test_from_a_new_thread():
    """A thread whose first CUDA work is the product (as autograd's threads)."""
    import threading
    g = gen(21)
    plan = make_plan([300, 0, 200])
    x, w = randn(g, 500, 128, dtype=torch.bfloat16), randn(g, 3, 128, 256, dtype=torch.bfloat16)
    q, s = E.quantize_rows(x)
    wq, ws = E.quantize_experts(w)
    dy = randn(g, 500, 256, dtype=torch.bfloat16)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    y = E.grouped_matmul(*leaves, plan)
    want = (E.grouped_matmul(x, w, plan), E.int8_matmul(q, s, wq, ws, plan),
            *torch.autograd.grad(y, leaves, dy, retain_graph=True))
    torch.cuda.synchronize()
    for i, f in enumerate((lambda: E.grouped_matmul(x, w, plan), lambda: E.int8_matmul(q, s, wq, ws, plan),
                           lambda: torch.autograd.grad(y, leaves[:1], dy, retain_graph=True)[0],
                           lambda: torch.autograd.grad(y, leaves[1:], dy, retain_graph=True)[0])):
        got = []
        f()  # its buffers are in the allocator's cache afterwards
        thread = threading.Thread(target=lambda: got.append(f()))
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert got and torch.equal(got[0], want[i])


def test_same_bits_twice():
    """No result depends on the schedule."""
    plan = make_plan([40, 3, 900, 16, 0, 1], 2)
    g = gen(19)
    x = randn(g, plan.num_tokens, 1024, dtype=torch.bfloat16).requires_grad_()
    w = randn(g, 6, 1024, 264, dtype=torch.bfloat16).requires_grad_()
    dy = randn(g, plan.num_rows, 264, dtype=torch.bfloat16)
    runs = []
    for _ in range(3):
        y = E.grouped_matmul(x, w, plan, gather=True)
        runs.append((y, *torch.autograd.grad(y, (x, w), dy)))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)
