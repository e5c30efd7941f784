"""8-bit floating-point rounding and products on the GPU against plain implementations in 64 bits.

Bounds, from the arithmetic: rounding to 8 bits is exact to compare (the scale is a
power of two). A product's sum runs over blocks of 128 in the tensor cores and over the
blocks in fp32: each step is off by at most 2^-23 of the magnitudes so far (truncation
included), the two scales' product and its multiplication by 2^-24 each, so
``(128 + blocks + 3) * 2**-23`` of the terms' magnitudes, far less in the 2-norm; the
result is rounded once."""

import math

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L
from test_gpu_experts import SIZES, TINY, TYPES, UNIT, gen, make_plan, randn
from test_gpu_gated import ACTS, act_error, act_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def scale_ref(peak):
    """The smallest power of two with peak <= 448 s, at least 2^-126, in 64 bits."""
    m, e = torch.frexp(peak.double())
    return torch.ldexp(torch.ones_like(m), torch.where(peak > 0, (e - 9 + (m > 0.875).int()), -126).clamp(min=-126))


def round_ref(v):
    """v (64 bits, |v| <= 448) to the nearest e4m3, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def quantize_ref(x):
    R, K = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -K % 128)).reshape(R, blocks(K), 128)
    s = scale_ref(b.abs().amax(2))
    return round_ref(b / s[..., None]).reshape(R, blocks(K) * 128)[:, :K], s


def spread(s, n, k):
    return s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


@pytest.mark.parametrize("R,K", [(1, 1), (3, 8), (5, 128), (2, 129), (17, 1000), (64, 4096), (7, 1025), (300, 136),
                                 (1, 70000), (2, 0), (0, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize(R, K, dtype):
    g = gen(R * K)
    x = randn(g, R, K, dtype=dtype)
    if R:
        x = (x.float() * torch.exp2(torch.randint(-12, 12, (R, 1), generator=g, device=DEV))).to(dtype)
    q, s = E.quantize_blocks(x)
    assert q.dtype == E4M3 and s.dtype == torch.float32 and q.shape == (R, K) and s.shape == (R, blocks(K))
    rq, rs = quantize_ref(x)
    assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_quantize_every_value(dtype):
    """Every finite 16-bit value, each beside a largest one that does and does not set a new power of two."""
    v = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[v.isfinite()]
    v = torch.cat([v, v.new_zeros(-v.numel() % 127)]).reshape(-1, 127)
    for top in (1.0, 1.75, 1.7578125, 1.9921875, 3.0e4):
        x = torch.cat([torch.full_like(v[:, :1], top), v], 1)
        q, s = E.quantize_blocks(x)
        rq, rs = quantize_ref(x)
        assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq)


def test_quantize_special():
    x = torch.zeros(6, 256, device=DEV)
    x[1, 3], x[2, 200], x[3, 7] = math.inf, math.nan, torch.finfo(torch.float32).max
    x[4, :4] = torch.tensor([1e-45, 2.0 ** -130, -2.0 ** -118, 2.0 ** -127], device=DEV)
    x[5, 0], x[5, 1] = 448.0, 448.0 * 2 ** -15
    q, s = E.quantize_blocks(x)
    assert bool(q[1, :128].isnan().all()) and bool(s[1, 0].isnan()) and not q[1, 128:].float().any()
    assert bool(q[2, 128:].isnan().all()) and bool(s[2, 1].isnan()) and not s[2, 0].isnan()
    rest = [0, 3, 4, 5]
    rq, rs = quantize_ref(x[rest])
    assert torch.equal(q[rest].double(), rq) and torch.equal(s[rest].double(), rs)
    assert float(s[0, 0]) == 2.0 ** -126 and float(s[5, 0]) == 1.0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_activation(act, dtype):
    """The rounded product of activation and up; where it is next to a border, either side."""
    g = gen(5)
    for R, K in ((40, 512), (9, 131)):
        x = randn(g, R, 2 * K, dtype=dtype, scale=3.0)
        q, s = E.quantize_blocks(x, activation=act)
        assert q.shape == (R, K)
        gate, up = x[:, :K].double(), x[:, K:].double()
        f = act_ref(act, gate)[0]
        h, off = f * up, (act_error(gate) * f.abs() + 1e-37) * up.abs() + 2.0 ** -24 * (f * up).abs()
        got = q.double() * s.double().repeat_interleave(128, 1)[:, :K]
        step = s.double().repeat_interleave(128, 1)[:, :K] * torch.exp2(
            torch.floor(torch.log2((h.abs() / s.double().repeat_interleave(128, 1)[:, :K]).clamp(min=2.0 ** -6))) - 3)
        assert bool(((got - h).abs() <= step / 2 + off).all())
        peak = torch.nn.functional.pad(h.abs(), (0, -K % 128)).reshape(R, -1, 128).amax(2)
        least = s == 2.0 ** -126  # a block of zeros
        assert bool((peak * (1 - 1e-5) <= 448 * s).all()) and bool(((peak * (1 + 1e-5) > 224 * s) | least).all())


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (200, 300), (3, 130, 257), (2, 2, 64, 40), (0, 8, 8), (5, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_weights(shape, dtype):
    g = gen(len(shape))
    w = randn(g, *shape, dtype=dtype)
    q, s = E.quantize_block_weights(w)
    K, N = shape[-2:]
    assert q.shape == (*shape[:-2], N, K) and s.shape == (*shape[:-2], blocks(N), blocks(K))
    if not w.numel():
        return
    t = w.double().transpose(-1, -2).reshape(-1, N, K)
    p = torch.nn.functional.pad(t, (0, -K % 128, 0, -N % 128)).reshape(t.shape[0], blocks(N), 128, blocks(K), 128)
    rs = scale_ref(p.abs().amax((2, 4)))
    assert torch.equal(s.double().reshape(rs.shape), rs)
    assert torch.equal(q.double().reshape(t.shape), round_ref(t / spread(rs, N, K)))


def random8(g, *shape):
    """e4m3 values over a few powers of two, and some zeros."""
    v = torch.randn(*shape, generator=g, device=DEV) * torch.exp2(torch.randint(-3, 6, shape, generator=g, device=DEV))
    return v.to(E4M3)


def scales(g, *shape):
    """Scales that are no powers of two, of either sign."""
    return torch.randn(*shape, generator=g, device=DEV) * 0.01


def operands(g, R, N, K, experts=()):
    return (random8(g, R, K), scales(g, R, blocks(K)), random8(g, *experts, N, K),
            scales(g, *experts, blocks(N), blocks(K)))


def product_ref(q, s, wq, ws, plan=None, gather=False):
    """(y, magnitudes) in 64 bits."""
    x = q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    w = wq.double() * spread(ws, *wq.shape[-2:])
    if plan is None:
        return x @ w.t(), x.abs() @ w.abs().t()
    y = x.new_zeros(plan.num_rows, w.shape[1])
    m = torch.zeros_like(y)
    off, order = plan.offsets.tolist(), plan.order.long()
    for e in range(plan.num_experts):
        r = slice(off[e], off[e + 1])
        a = x[order[r] // plan.top_k] if gather else x[r]
        y[r], m[r] = a @ w[e].t(), a.abs() @ w[e].abs().t()
    return y, m


def check(got, ref, mag, K, dtype):
    assert got.dtype == dtype and got.shape == ref.shape
    err = (got.double() - ref).abs()
    over = err - (UNIT[dtype] * ref.abs() + (128 + blocks(K) + 3) * 2.0 ** -23 * mag + TINY[dtype])
    assert bool((over <= 0).all()), float(over.max())
    if ref.numel() > 500:
        assert float(err.norm()) <= (UNIT[dtype] + 2.0 ** -19) * float(ref.norm())
    E.check_device_errors()


@pytest.mark.parametrize("R", [1, 3, 16, 33, 127, 129, 300, 700])
@pytest.mark.parametrize("K,N", [(16, 8), (128, 128), (1040, 264), (100, 37), (4096, 1000), (5, 3), (384, 4000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_dense(R, K, N, dtype):
    args = operands(gen(R + K), R, N, K)
    check(E.fp8_matmul(*args, out_dtype=dtype), *product_ref(*args), K, dtype)


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N", [(64, 128), (16, 8), (400, 72), (37, 101), (272, 520)])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(sizes, K, N, gather):
    s = SIZES[sizes]
    k = 2 if sum(s) % 2 == 0 else 1
    plan = make_plan(s, k, dropped=3 * k, seed=K)
    args = operands(gen(K + N), plan.num_tokens if gather else plan.num_rows, N, K, (len(s),))
    for dtype in TYPES:
        y = E.fp8_matmul(*args, plan, gather=gather, out_dtype=dtype)
        check(y, *product_ref(*args, plan, gather), K, dtype)
        assert not y[sum(s):].any()


LONG = [200, 701, 256, 0, 513, 390, 128, 511, 257]         # a mean past 128 rows
SHORT = [10 + 37 * i % 91 for i in range(58)] + [0, 129]   # 10 to 100 rows, none, and a tile and one


@pytest.mark.parametrize("sizes,K,N,path", [
    (LONG, 400, 2064, L.ES_GROUPED_WIDE), (LONG, 528, 2061, L.ES_GROUPED_WIDE), (LONG, 136, 2200, L.ES_GROUPED_WIDE),
    (SHORT, 400, 1032, L.ES_GROUPED_NARROW), (SHORT, 1100, 333, L.ES_GROUPED_NARROW),
    ([5], 4096, 1000, L.ES_GROUPED_SPLIT), ([130, 7], 2100, 264, L.ES_GROUPED_SPLIT), ([128], 1024, 4096,
                                                                                     L.ES_GROUPED_SPLIT)])
@pytest.mark.parametrize("dtype", TYPES)
def test_shapes(sizes, K, N, path, dtype):
    """Every tile shape, with ragged groups, several tiles a CTA, last tiles of rows and channels."""
    plan = make_plan(sizes, 1, dropped=4)
    assert L.lib().es_fp8_matmul_path(len(sizes), K, N, plan.num_rows) == path
    args = operands(gen(N), plan.num_rows, N, K, (len(sizes),))
    y = E.fp8_matmul(*args, plan, out_dtype=dtype)
    check(y, *product_ref(*args, plan), K, dtype)
    assert not y[sum(sizes):].any()


def test_long_sums():
    """Sums of one sign, past any one chain: no drift beyond a block's."""
    g = gen(3)
    for R, K, N in ((20, 65536, 128), (300, 32768, 8200)):
        q = (torch.rand(R, K, generator=g, device=DEV) * 8 + 1).to(E4M3)
        wq = (torch.rand(N, K, generator=g, device=DEV) * 8 + 1).to(E4M3)
        s, ws = torch.full((R, K // 128), 0.3, device=DEV), torch.full((blocks(N), K // 128), 0.7, device=DEV)
        y = E.fp8_matmul(q, s, wq, ws, out_dtype=torch.float32)
        n = min(N, 512)
        ref = (q.double() @ wq[:n].double().t()) * float(s[0, 0].double()) * float(ws[0, 0].double())
        # of one sign: the mean over a block's 128 truncations, at most 2^-24 of the sum each, half of them on average,
        # and the roundings of K / 128 additions, which are to nearest
        assert float(((y[:, :n].double() - ref) / ref).abs().max()) <= (64 + K / 128 / 8) * 2.0 ** -24


def test_extreme_scales():
    """Scales whose product is past the type's ends, with sums that bring the result back."""
    cases = [(2.0 ** 100, 2.0 ** 100, 0.0), (2.0 ** 66, 2.0 ** 66, 2.0 ** -18), (2.0 ** -100, 2.0 ** -40, 448.0 * 448),
             (2.0 ** -126, 2.0 ** 120, 2.0 ** -18), (2.0 ** -80, 2.0 ** -60, 3.0), (2.0 ** 127, 2.0 ** -126, 5.0),
             (1e38, 100.0, 2.0 ** -18), (0.0, 1e38, 448.0)]
    for xs, ws, v in cases:
        q = torch.zeros(1, 128, device=DEV)
        wq = torch.zeros(1, 128, device=DEV)
        if v == 2.0 ** -18:
            q[0, 0], wq[0, 0] = 2.0 ** -9, 2.0 ** -9
        elif v == 448.0 * 448:
            q[0, 0], wq[0, 0] = 448.0, 448.0
        else:
            q[0, 0], wq[0, 0] = v, 1.0
        a, b = torch.full((1, 1), xs, device=DEV), torch.full((1, 1), ws, device=DEV)
        y = float(E.fp8_matmul(q.to(E4M3), a, wq.to(E4M3), b, out_dtype=torch.float32))
        want = float(q.to(E4M3).double()[0, 0] * wq.to(E4M3).double()[0, 0]) * float(a.double()) * float(b.double())
        want32 = float(torch.tensor(want, dtype=torch.float64).float())
        assert y == want32 or abs(y - want) <= 2.0 ** -23 * abs(want) + 2.0 ** -149, (xs, ws, v, y, want)


@pytest.mark.parametrize("sizes", [[5, 3], [150, 200], [700, 900]])
def test_nan_stays_alone(sizes):
    plan = make_plan(sizes, 1, dropped=2)
    n, N, K = sum(sizes), 1000, 300
    q, s, wq, ws = operands(gen(1), plan.num_rows, N, K, (2,))
    clean = E.fp8_matmul(q, s, wq, ws, plan)
    q, s, wq = q.float(), s.clone(), wq.float()
    q[1, 5], s[2, 1], wq[1, 7, 9] = math.nan, math.inf, math.nan
    q[n:], s[n:] = math.nan, math.nan
    got = E.fp8_matmul(q.to(E4M3), s, wq.to(E4M3), ws, plan)
    assert bool(got[1].isnan().all()) and not bool(got[2].isfinite().any())
    assert bool(got[sizes[0]:n, 7].isnan().all())
    rows = [r for r in range(plan.num_rows) if r not in (1, 2)]
    cols = [c for c in range(N) if c != 7]
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    assert torch.equal(got[0], clean[0])


def test_layouts():
    g = gen(2)
    plan = make_plan([70, 0, 33], 1)
    q, s, wq, ws = operands(g, 103, 136, 272, (3,))
    want = E.fp8_matmul(q, s, wq, ws, plan)

    def same(*args):
        assert torch.equal(E.fp8_matmul(*args, plan), want)

    wide = torch.zeros(103, 320, device=DEV).to(E4M3)
    for at in (0, 16, 5):
        wide.view(torch.uint8)[:, at:at + 272] = q.view(torch.uint8)
        same(wide[:, at:at + 272], s, wq, ws)
    big = torch.zeros(3, 136, 300, device=DEV).to(E4M3)
    for at in (0, 3):
        big.view(torch.uint8)[:, :, at:at + 272] = wq.view(torch.uint8)
        same(q, s, big[:, :, at:at + 272], ws)
    same(q, s.t().contiguous().t(), wq, ws.transpose(1, 2).contiguous().transpose(1, 2))
    same(q, s, wq.transpose(0, 1).contiguous().transpose(0, 1), ws)
    first = E.fp8_matmul(q, s, wq[:1].expand(3, 136, 272), ws, plan)
    assert torch.equal(first[:70], want[:70])


def test_quantized_product():
    """Rounded operands as a program makes them, against the exact product: 8 bits' own error, 2^-4 a value at most."""
    g = gen(8)
    x, w = randn(g, 200, 1024, dtype=torch.bfloat16), randn(g, 1024, 384, dtype=torch.bfloat16)
    y = E.fp8_matmul(*E.quantize_blocks(x), *E.quantize_block_weights(w), out_dtype=torch.float32)
    ref = x.double() @ w.double()
    # half a step is at most 2^-4 of a value, a third of that in the mean square, for each operand
    assert float((y.double() - ref).norm()) <= 2 * 2.0 ** -4 / math.sqrt(3) * float(ref.norm())


def test_streams_graph_thread():
    import threading
    g = gen(9)
    plan = make_plan([40, 0, 300, 16], 2)
    x = randn(g, plan.num_tokens, 512, dtype=torch.bfloat16)
    wq, ws = E.quantize_block_weights(randn(g, 4, 512, 264))

    def step():
        return E.fp8_matmul(*E.quantize_blocks(x), wq, ws, plan, gather=True)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    x.mul_(-2)
    graph.replay()
    assert torch.equal(kept, step()) and torch.equal(kept, -2 * want)
    out = []
    thread = threading.Thread(target=lambda: out.append(step()))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(out[0], kept)
    E.check_device_errors()


def test_empty():
    for R, K, N in ((0, 128, 8), (4, 0, 8), (4, 128, 0)):
        x, w = torch.ones(R, K, device=DEV), torch.ones(K, N, device=DEV)
        y = E.fp8_matmul(*E.quantize_blocks(x), *E.quantize_block_weights(w))
        assert y.shape == (R, N) and not y.any()
    plan = make_plan([0, 0], 1, dropped=5)
    x, w = torch.full((5, 64), math.nan, device=DEV), torch.ones(2, 64, 72, device=DEV)
    assert not E.fp8_matmul(*E.quantize_blocks(x), *E.quantize_block_weights(w), plan).any()


def test_refusals():
    x, w = torch.zeros(4, 256, device=DEV), torch.zeros(256, 130, device=DEV)
    (q, s), (wq, ws) = E.quantize_blocks(x), E.quantize_block_weights(w)
    plan = make_plan([3, 1], 1)
    for call in (lambda: E.fp8_matmul(q[:, :200], s, wq, ws), lambda: E.fp8_matmul(q, s[:, :1], wq, ws),
                 lambda: E.fp8_matmul(q, s, wq, ws[:1]), lambda: E.fp8_matmul(q, s, wq, ws, plan),
                 lambda: E.fp8_matmul(q, s, wq, ws, gather=True), lambda: E.fp8_matmul(q, s[:3], wq, ws),
                 lambda: E.quantize_blocks(x[0]), lambda: E.quantize_blocks(x[:, :255], activation="silu"),
                 lambda: E.quantize_blocks(x, activation="swish"), lambda: E.quantize_blocks(x.cpu()),
                 lambda: E.quantize_block_weights(w[0]), lambda: E.fp8_matmul(q, s.cpu(), wq, ws),
                 lambda: E.fp8_matmul(q, s, wq[None].expand(2, 130, 256), ws[None].expand(3, 2, 2), plan)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: E.fp8_matmul(x, s, wq, ws), lambda: E.fp8_matmul(q, s.half(), wq, ws),
                 lambda: E.fp8_matmul(q, s, wq, ws, out_dtype=torch.float64), lambda: E.quantize_blocks(x.double()),
                 lambda: E.quantize_block_weights(w.double()), lambda: E.fp8_matmul(q, s, wq, ws, 3)):
        with pytest.raises(TypeError):
            call()
    x.requires_grad_()
    assert not E.quantize_blocks(x)[1].requires_grad


def test_quantize_past_32_bits():
    """More values than 32 bits number."""
    R, K = 70001, 32768
    x = torch.zeros(R, K, dtype=torch.bfloat16, device=DEV)
    x[-2:] = randn(gen(4), 2, K, dtype=torch.bfloat16)
    q, s = E.quantize_blocks(x)
    rq, rs = quantize_ref(x[-2:])
    assert torch.equal(q[-2:].double(), rq) and torch.equal(s[-2:].double(), rs)
    assert not q[:-2].view(torch.uint8).any()


def test_output_past_32_bits():
    """An output of more than 2^31 values, and rows of a group behind that border."""
    R, K, N = 300000, 64, 8192
    g = gen(6)
    plan = make_plan([R - 200, 200], 1)
    q, s, wq, ws = operands(g, R, N, K, (2,))
    y = E.fp8_matmul(q, s, wq, ws, plan)
    ref = (q[-200:].double() * s[-200:].double()) @ (wq[1].double() * spread(ws[1], N, K)).t()
    mag = (q[-200:].double() * s[-200:].double()).abs() @ (wq[1].double() * spread(ws[1], N, K)).abs().t()
    check(y[-200:], ref, mag, K, torch.bfloat16)


# What a row's blocks of depth hold, eight blocks (the kernel's unit) at a time: ordinary values; zeros with the least scale;
# products of scales below fp32's normal numbers; above its largest, over zeros and over the smallest values.
PLAIN, ZERO, TINY_SCALES, OVER_ZERO, OVER_SMALL = range(5)


def mixed_rows(g, R, K, kinds):
    """(q, scale) with rows that hold, from one eight blocks to the next, every order of ``kinds``."""
    n = blocks(K)
    kind = (torch.arange(R, device=DEV)[:, None] // len(kinds) ** torch.arange(-(-n // 8), device=DEV)) % len(kinds)
    kind = torch.tensor(kinds, device=DEV)[kind].repeat_interleave(8, 1)[:, :n]
    q, s = random8(g, R, n, 128).float(), scales(g, R, n)
    small = torch.zeros_like(q)
    small[..., 5] = 2.0 ** -9
    q = torch.where((kind == PLAIN)[..., None] | (kind == TINY_SCALES)[..., None], q, 0.0)
    q = torch.where((kind == OVER_SMALL)[..., None], small, q)
    for k, v in ((ZERO, 2.0 ** -126), (TINY_SCALES, 2.0 ** -118), (OVER_ZERO, 3.0e38), (OVER_SMALL, 1.9 * 2.0 ** 107)):
        s = torch.where(kind == k, v, s)
    return q.reshape(R, n * 128)[:, :K].to(E4M3).contiguous(), s


@pytest.mark.parametrize("R,K,N,path", [
    (625, 2500, 10000, L.ES_GROUPED_WIDE), (125, 2304, 19000, L.ES_GROUPED_NARROW),
    (25, 12100, 300, L.ES_GROUPED_SPLIT), (125, 2200, 9000, L.ES_GROUPED_SPLIT)])
@pytest.mark.parametrize("kinds", [(PLAIN, ZERO, TINY_SCALES), (PLAIN, ZERO, OVER_ZERO),
                                   (PLAIN, ZERO, TINY_SCALES, OVER_ZERO, OVER_SMALL)])
def test_scales_change_along_the_depth(R, K, N, path, kinds):
    """Blocks whose scales' products are past fp32's ends before, between and after ordinary ones: each counts as what it
    is. Each block's term is within the usual few roundings of its magnitude, or within what it loses at fp32's lower end:
    less than 2^-150, and beside a product of scales of 2^36 or more, which is held times 2^-40, half a unit of
    2^(-149 + 40) times a sum of 128 products of up to 2^17.7, 2^-85.3."""
    g = gen(K)
    assert L.lib().es_fp8_matmul_path(0, K, N, R) == path
    q, s = mixed_rows(g, R, K, kinds)
    wq = random8(g, N, K).float().clamp(-16, 16).to(E4M3)
    ws = torch.exp2(20.0 * torch.randint(-1, 2, (blocks(N), blocks(K)), generator=g, device=DEV)) \
        * (1 + torch.rand(blocks(N), blocks(K), generator=g, device=DEV))
    y = E.fp8_matmul(q, s, wq, ws, out_dtype=torch.float32)
    ref, mag = product_ref(q, s, wq, ws)
    assert float(ref.abs().max()) < torch.finfo(torch.float32).max / 2  # every result is a number
    large = ((s.double()[:, None] * ws.double()).abs().amax(2) >= 2.0 ** 36).repeat_interleave(128, 1)[:, :N]
    bound = UNIT[torch.float32] * ref.abs() + (128 + blocks(K) + 3) * 2.0 ** -23 * mag \
        + blocks(K) * (2.0 ** -150 + 2.0 ** -85 * large.double())
    assert bool(((y.double() - ref).abs() <= bound).all())
    E.check_device_errors()


@pytest.mark.parametrize("R", [3, 150, 700])
@pytest.mark.parametrize("act", [None, "relu"])
def test_quantized_blocks_of_zeros(R, act):
    """Zeros in x or in w, as the rounding makes them, behind and before sums above one."""
    g = gen(R)
    K, N = 2048 + 128, 3000
    x, w = randn(g, R, K if act is None else 2 * K, dtype=torch.bfloat16, scale=4.0), randn(g, K, N) * 0.02
    x[: R // 2, 1024:K] = 0  # of gate, with an activation
    x[R // 2:, :1024] = 0
    w[1500:, :200] = 0
    q, s = E.quantize_blocks(x, activation=act)
    wq, ws = E.quantize_block_weights(w)
    ref, mag = product_ref(q, s, wq, ws)
    assert float(ref.abs().max()) > 4
    check(E.fp8_matmul(q, s, wq, ws, out_dtype=torch.float32), ref, mag, K, torch.float32)


@pytest.mark.parametrize("R", [40, 700])
def test_a_row_has_its_bits_beside_any_others(R):
    """A row's result does not depend on what scales the rows beside it have."""
    g = gen(R + 1)
    q, s, wq, ws = operands(g, R, 9000, 2200)
    ws = ws.abs() + 0.001
    y = E.fp8_matmul(q, s, wq, ws)
    s2 = s.clone()
    s2[1::2, 3::4] = 2.0 ** -126
    s2[2::8, 5] = 3.0e38
    z = E.fp8_matmul(q, s2, wq, ws)
    same = (s == s2).all(1)
    assert torch.equal(y[same], z[same])
