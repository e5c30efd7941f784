"""Expert operators on the GPU at the ends of their types, of their depths and of their tile shapes.

Bounds are derived as in ``test_gpu_experts``: one rounding of the result's
type, and for fp32 sums ``2**-23`` of the products' magnitudes a step, in the
2-norm over many values at most ``2**-19``.
"""

import math
import threading

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L
from test_gpu_experts import TYPES, UNIT, check_int8, gen, grouped_ref, int8_ref, int8s, make_plan, near, randn

pytestmark = pytest.mark.gpu

DEV = "cuda"


def same_kinds(got, ref):
    """The infinities and NaN of got are those of ref (64 bits); where ref is finite the two are near."""
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.isposinf(), ref.isposinf()) and torch.equal(got.isneginf(), ref.isneginf())
    there = ref.isfinite()
    err = (got.double() - ref)[there].norm()
    assert float(err) <= (UNIT[got.dtype] + 2.0 ** -19) * float(ref[there].norm())


# ----------------------------------------- infinities and the largest values, fp32

@pytest.mark.parametrize("sizes", [[3, 0, 2], [130, 0, 70], [700, 500, 300]])
@pytest.mark.parametrize("K,N", [(96, 64), (1100, 132), (72, 2060)])
@pytest.mark.parametrize("transposed", [False, True])
def test_grouped_infinite(sizes, K, N, transposed):
    """An infinity in fp32 is what fp32 arithmetic makes of it, whatever the length of its group."""
    plan = make_plan(sizes, 1, dropped=2)
    g = gen(K + N)
    x = randn(g, plan.num_rows, K)
    w = randn(g, 3, K, N, scale=K ** -0.5)
    dy = randn(g, plan.num_rows, N)
    off = plan.offsets.tolist()
    w[0, 5, 3] = 0.0
    x[1, 5], x[off[2], K - 1], x[off[2] + 1, 0] = math.inf, -math.inf, math.nan
    w[2, 7, N - 1], w[2, 8, N - 1] = math.inf, -math.inf
    dy[2, 1], dy[off[2] + 1, N - 2] = -math.inf, math.inf
    dy[off[2], N - 1] = 0.0
    if transposed:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x.requires_grad_()
    w.requires_grad_()
    y = E.grouped_matmul(x, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, _, rx, _, rw, _ = grouped_ref(x, w, plan, False, dy)
    for got, ref in ((y.detach(), ry), (dx, rx), (dw, rw)):
        assert bool(ref.isinf().any()) and bool(ref.isnan().any())
        same_kinds(got, ref)


@pytest.mark.parametrize("sizes", [[3, 2], [130, 70], [700, 500]])
@pytest.mark.parametrize("N", [8, 2060])
def test_grouped_largest(sizes, N):
    """Values and products next to the type's largest stay finite, though their first planes are rounded up."""
    big = torch.finfo(torch.float32).max
    plan = make_plan(sizes, 1)
    g = gen(N)
    K = 72
    x = randn(g, plan.num_rows, K) * 2.0 ** -10
    w = randn(g, 2, K, N)
    w[0, 3, 2], w[1, K - 1, N - 1] = big, -big
    x[1], w[0, :, 5] = 0.0, 0.0
    x[1, 3], w[0, 3, 5] = 3.385e38, 1.0045  # both planes round up: their product is past the largest value
    x[1, 4], w[0, 4, 2] = 0.0, 0.0
    w[0, 3, 2] = 0.9
    w[0, 4, 3] = big
    w[0, 3, torch.arange(N, device=DEV) > 5] = 0.0
    w[0, 3, :2] = 0.5
    w[0, 3, 3:5] = -1.0
    y = E.grouped_matmul(x, w, plan)
    ry, my = grouped_ref(x, w, plan, False)[:2]
    assert bool(ry.abs().max() < big) and bool(ry.abs().max() > 0.999 * big)
    near(y / 2.0 ** 64, ry / 2.0 ** 64, my / 2.0 ** 64, K, torch.float32)


@pytest.mark.parametrize("K,N", [(260, 132), (2520, 68), (8, 200)])
@pytest.mark.parametrize("transposed", [False, True])
def test_grouped_few_rows_all_infinite(K, N, transposed):
    """Every row of several tiles holds an infinity, or a NaN beside it, or the weights do."""
    sizes = [19, 0, 7, 16, 1]
    plan = make_plan(sizes, 1)
    g = gen(K)
    x, w = randn(g, plan.num_rows, K), randn(g, 5, K, N, scale=K ** -0.5)
    rows = torch.arange(plan.num_rows, device=DEV)
    x[rows, rows % K] = math.inf * (1 - 2 * (rows % 2).float())
    x[rows[::5], (rows[::5] + 3) % K] = math.nan
    x[4] = 0.0
    w[0, :, 7], w[2, 1, N - 1], w[3, K - 1, ::3] = 0.0, math.nan, math.inf
    if transposed:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    y = E.grouped_matmul(x, w, plan)
    same_kinds(y, grouped_ref(x, w, plan, False)[0])


def test_grouped_few_rows_poisoned_time():
    """Rows that are NaN take about the time of rows that are not."""
    plan = make_plan([8] * 12, 1)
    g = gen(1)
    w = randn(g, 12, 2048, 1024)
    clean = randn(g, 96, 2048)
    bad = torch.full_like(clean, math.nan)

    def microseconds(x):
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                E.grouped_matmul(x, w, plan)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 100)
        return best

    microseconds(clean)
    assert microseconds(bad) <= 2 * microseconds(clean)


# ----------------------------------------------------------- long sums of one sign

def positive(g, *shape, dtype, scale=1.0):
    return (torch.rand(*shape, generator=g, device=DEV) * scale).to(dtype)


def unbiased(got, ref, n):
    """Positive sums of n products. Where they are rounded once, to nearest, the mean error over many is a small part
    of the rounding's unit; a third leaves room for an accumulator that truncates."""
    near(got, ref, ref, n, got.dtype)
    unit = max(UNIT[got.dtype], 2.0 ** -19)
    assert abs(float(((got.double() - ref) / ref).mean())) <= unit / 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[131072, 300], [16384, 0, 16385, 70000], [7, 20000, 65536, 3]])
@pytest.mark.parametrize("transposed", [False, True])
def test_long_groups_weights_gradient(dtype, sizes, transposed):
    plan = make_plan(sizes, 1, dropped=5)
    g = gen(len(sizes))
    K, N = 40, 23 if transposed else 136
    x = positive(g, plan.num_rows, K, dtype=dtype)
    w = torch.zeros(len(sizes), *((N, K) if transposed else (K, N)), dtype=dtype, device=DEV)
    w = (w.transpose(1, 2) if transposed else w).requires_grad_()
    dy = positive(g, plan.num_rows, N, dtype=dtype, scale=2.0 ** -6)
    dw, = torch.autograd.grad(E.grouped_matmul(x, w, plan), w, dy)
    off = plan.offsets.tolist()
    for e, n in enumerate(sizes):
        r = slice(off[e], off[e + 1])
        if n:
            unbiased(dw[e], x[r].double().t() @ dy[r].double(), n)
        else:
            assert not dw[e].any()


@pytest.mark.parametrize("dtype,K", [(torch.float16, 20000), (torch.float16, 16384), (torch.bfloat16, 66000),
                                     (torch.float32, 20000)])
@pytest.mark.parametrize("sizes,N", [([30], 9608), ([5, 0, 2], 136), ([700], 12301)])
@pytest.mark.parametrize("transposed", [False, True])
def test_deep_rows(dtype, K, sizes, N, transposed):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    plan = make_plan(sizes, 1, dropped=1)
    g = gen(N)
    x = positive(g, plan.num_rows, K, dtype=dtype)
    w = positive(g, len(sizes), *((N, K) if transposed else (K, N)), dtype=dtype, scale=2.0 ** -6)
    w = w.transpose(1, 2) if transposed else w
    y = E.grouped_matmul(x, w, plan)
    off = plan.offsets.tolist()
    for e in range(len(sizes)):
        if sizes[e]:
            r = slice(off[e], off[e + 1])
            unbiased(y[r], x[r].double() @ w[e].double(), K)
    assert not y[off[-1]:].any()


# --------------------------------------------------------------- 8-bit scales

@pytest.mark.parametrize("rows,N", [(3, 40), (70, 1000), (700, 5000)])
@pytest.mark.parametrize("grouped", [False, True])
def test_int8_scales_of_any_size(rows, N, grouped):
    """Large scales of rows and small ones of channels, or the reverse: finite products stay finite."""
    g = gen(rows + N)
    K = 1040
    plan = make_plan([rows // 3, 0, rows - rows // 3], 1) if grouped else None
    q, wq = int8s(g, rows, K), int8s(g, *((3, N, K) if grouped else (N, K)))
    q[0], wq[..., 0, :], wq[..., 1, :] = 127, -127, 0  # the largest sum, and sums of zero
    for big, small in ((3e35, 1e-35), (1e-37, 3e33), (2e15, 1e14), (1e-19, 1e-18)):
        s, ws = ((1 + torch.rand(*shape, generator=g, device=DEV)) * scale
                 for shape, scale in (((rows,), big), (wq.shape[:-1], small)))
        y = E.int8_matmul(q, s, wq, ws, plan, out_dtype=torch.float32)
        ref = int8_ref(q, s, wq, ws, plan, False)
        assert bool(((ref.abs() > 2e-38) & (ref.abs() < 3.4e38) | (ref == 0)).all())
        check_int8(y, ref, torch.float32)


# ------------------------------------------------------------------- empty weights

@pytest.mark.parametrize("shape", [(3, 0, 5), (0, 4, 5), (3, 4, 0), (0, 0), (7, 0), (0, 7)])
def test_quantize_experts_empty(shape):
    q, s = E.quantize_experts(torch.zeros(shape, device=DEV))
    assert q.dtype == torch.int8 and q.shape == (*shape[:-2], shape[-1], shape[-2])
    assert s.dtype == torch.float32 and s.shape == (*shape[:-2], shape[-1]) and not s.any()


# ------------------------------------------------------------- derivatives refused

@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(leaf):
    """A tangent raises instead of being dropped, in an operand and in a gradient; a level without one changes nothing."""
    import torch.autograd.forward_ad as fw
    plan = make_plan([3, 5], 2)
    g = gen(1)
    logits, x, w = randn(g, 4, 2), randn(g, 4, 16), randn(g, 2, 16, 8)
    y, weights, router = randn(g, 8, 16), torch.rand(4, 2, generator=g, device=DEV), randn(g, 16, 2)
    calls = ((lambda a: E.route_experts(a, 2)[0], [logits]), (lambda a, b: E.grouped_matmul(a, b, plan, True), [x, w]),
             (lambda a, b: E.combine_experts(a, b, plan), [y, weights]),
             (lambda a, b: E.expert_mlp(a, b, randn(gen(2), 2, 16, 32), randn(gen(2), 2, 16, 16), 2), [x, router]))
    for call, args in calls:
        args = [a.detach().requires_grad_(leaf) for a in args]
        want = call(*args)
        with fw.dual_level():
            assert torch.equal(call(*args), want)
            for i in range(len(args)):
                duals = list(args)
                duals[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    call(*duals)
            if leaf:
                out = call(*args)
                with pytest.raises(NotImplementedError):
                    torch.autograd.grad(out, args, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("leaf", ["x", "router"])
def test_gradient_through_8_bits_is_refused(leaf):
    """The 8-bit layer serves operands that require a gradient, and gives none of it instead of a part."""
    g = gen(3)
    x, router = randn(g, 10, 16), randn(g, 16, 4)
    w_in, w_out = E.quantize_experts(randn(g, 4, 16, 32)), E.quantize_experts(randn(g, 4, 16, 16))
    want = E.expert_mlp(x, router, w_in, w_out, 2)
    assert not want.requires_grad
    (x if leaf == "x" else router).requires_grad_()
    with torch.no_grad():
        assert torch.equal(E.expert_mlp(x, router, w_in, w_out, 2), want)
    out = E.expert_mlp(x, router, w_in, w_out, 2)
    assert torch.equal(out.detach(), want)
    for loss in (out.sum(), (x + out).sum()):
        with pytest.raises(RuntimeError, match="8-bit"):
            loss.backward(retain_graph=True)


# --------------------------------------------------------------------- threads

def test_plans_of_many_experts_from_threads():
    """Threads that order rows of different numbers of experts, whose kernels ask for different shared memory."""
    lib = L.lib()
    wanted = (1024, 690, 1000, 700)
    start = threading.Barrier(len(wanted))
    answers = []

    def calls(n):
        torch.cuda.set_device(0)
        e = torch.zeros(4, 1, dtype=torch.int32, device=DEV)
        off, order, position = (torch.empty(m, dtype=torch.int32, device=DEV) for m in (n + 1, 4, 4))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        args = (e.data_ptr(), 4, n, None, 0, off.data_ptr(), order.data_ptr(), position.data_ptr(), None,
                stream.cuda_stream)
        start.wait()
        got = {lib.es_expert_plan(*args) for _ in range(5000)}
        stream.synchronize()
        answers.append(got)

    threads = [threading.Thread(target=calls, args=(n,)) for n in wanted]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert answers == [{L.ES_OK}] * len(wanted)


# ------------------------------------------------------------------ captured calls

def test_replayed_failure_is_raised():
    """check_device_errors waits for the kernels of a replayed graph."""
    e = torch.zeros(10, 1, dtype=torch.int32, device=DEV)
    long = torch.zeros(8192, 8192, device=DEV)
    E.plan_experts(e, 4)
    E.check_device_errors()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(8):  # tens of milliseconds before the kernel that fails
            long @ long
        E.plan_experts(e, 4)
    E.check_device_errors()
    e[3] = 9
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
        with pytest.raises(ValueError, match="es_expert_plan"):
            E.check_device_errors()
    E.check_device_errors()
    del graph
