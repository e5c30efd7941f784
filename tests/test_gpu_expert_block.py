"""A layer of experts made of the gated products, the 8-bit floating-point products and the norms, as a program runs
them together: training steps against autograd in 64 bits, serving within its rounding, captured and replayed."""

import math

import pytest
import torch

import einjax_b200 as E
from test_gpu_experts import gen, randn
from test_gpu_gated import act_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def rms(v, w, eps):
    return v * w / (v.square().mean(1, keepdim=True) + eps).sqrt()


class _Act(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, name):
        a, s = act_ref(name, g)
        ctx.save_for_backward(s)
        return a

    @staticmethod
    def backward(ctx, d):
        return d * ctx.saved_tensors[0], None


def block_ref(p, act, k, scale, eps):
    """The block in 64 bits, differentiable."""
    x = p["x"]
    n = rms(x, p["norm_in"], eps) if "norm_in" in p else x
    top = torch.sort(n @ p["router"], dim=1, descending=True, stable=True)
    weights, experts = torch.softmax(top.values[:, :k], 1), top.indices[:, :k]
    y = torch.zeros_like(x)
    F = p["w_out"].shape[1]
    for e in range(p["w_in"].shape[0]):
        for j in range(k):
            at = (experts[:, j] == e).nonzero()[:, 0]
            h = n[at] @ p["w_in"][e]
            y = y.index_add(0, at, weights[at, j, None] * ((_Act.apply(h[:, :F], act) * h[:, F:]) @ p["w_out"][e]))
    if "norm_out" in p:
        y = rms(y, p["norm_out"], eps)
    if "gate" in p:
        y = y * p["gate"]
    return x + scale * y if scale is not None else y


def params(g, T, D, F, n, dtype, residual):
    p = {"x": randn(g, T, D), "router": randn(g, D, n, scale=2 * D ** -0.5),
         "w_in": randn(g, n, D, 2 * F, scale=D ** -0.5), "w_out": randn(g, n, F, D, scale=F ** -0.5)}
    if residual:
        p |= {"norm_in": 1 + randn(g, D, scale=0.2), "norm_out": 1 + randn(g, D, scale=0.2), "gate": randn(g, D)}
    return {k: v.to(dtype if k != "router" else torch.float32) for k, v in p.items()}


def call(p, k, act, scale):
    return E.expert_mlp(p["x"], p["router"], p["w_in"], p["w_out"], k, activation=act, norm_in=p.get("norm_in"),
                        norm_out=p.get("norm_out"), gate=p.get("gate"), scale=scale)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("residual", [False, True])
def test_training_fp32(act, residual):
    g = gen(len(act))
    p = params(g, 150, 64, 96, 6, torch.float32, residual)
    scale = 0.7 if residual else None
    for t in p.values():
        t.requires_grad_()
    out = call(p, 2, act, scale)
    dout = randn(g, 150, 64)
    got = torch.autograd.grad(out, list(p.values()), dout)
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    ref = block_ref(q, act, 2, scale, 1e-6)
    want = torch.autograd.grad(ref, list(q.values()), dout.double())
    for name, a, b in zip(("out", *p), (out.detach(), *got), (ref.detach(), *want)):
        # a chain of up to eight operators, each within 2^-18 in the norm, whose factors are of order one
        assert float((a.double() - b).norm()) <= 2.0 ** -14 * float(b.norm()), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_16_bits(dtype):
    g = gen(3)
    p = params(g, 700, 128, 192, 4, dtype, True)
    for t in p.values():
        t.requires_grad_()
    out = call(p, 2, "silu", 0.5)
    dout = randn(g, 700, 128, dtype=dtype)
    got = torch.autograd.grad(out, list(p.values()), dout)
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    # routed as the layer was: a tie of logits that rounding breaks is no error
    ref = block_ref(q, "silu", 2, 0.5, 1e-6)
    same = ((out.detach().double() - ref.detach()).norm(dim=1) <= 0.05 * ref.detach().norm(dim=1))
    assert float(same.double().mean()) > 0.98
    unit = torch.finfo(dtype).eps / 2
    err = (out.detach().double() - ref.detach())[same].norm() / ref.detach()[same].norm()
    assert float(err) <= 8 * unit  # x normalised, two products, the weighted sum and the result rounded: five roundings
    want = torch.autograd.grad(ref, list(q.values()), dout.double())
    for name, a, b in zip(p, got, want):
        # some twelve roundings in a chain, and the tokens whose routing differs (2% of the norm's square at most)
        assert float((a.double() - b).norm()) <= (16 * unit + 0.15) * float(b.norm()), name


def test_serving():
    g = gen(5)
    p = params(g, 300, 256, 384, 8, torch.bfloat16, True)
    ref = block_ref({k: v.double() for k, v in p.items()}, "silu", 2, 0.5, 1e-6)
    full = call(p, 2, "silu", 0.5)
    served = E.expert_mlp(p["x"], p["router"], E.quantize_block_weights(p["w_in"]), E.quantize_block_weights(p["w_out"]),
                          2, norm_in=p["norm_in"], norm_out=p["norm_out"], gate=p["gate"], scale=0.5)
    branch = (ref - p["x"].double()).norm()
    assert float((full.double() - ref).norm()) <= 0.05 * float(branch)
    # four operands rounded to 4 bits: half a step is up to 2^-4 of a value, 2^-4 / sqrt(3) in the mean square at the
    # very most, and all of them add up in squares
    assert float((served.double() - ref).norm()) <= (2 * 2.0 ** -4 / math.sqrt(3) * 2 ** 0.5 + 0.05) * float(branch)
    named = E.expert_mlp(p["x"], p["router"], E.quantize_block_weights(p["w_in"]), E.quantize_block_weights(p["w_out"]),
                         2, activation="silu", norm_in=p["norm_in"], norm_out=p["norm_out"], gate=p["gate"], scale=0.5)
    assert torch.equal(named, served)
    x = p["x"].clone().requires_grad_()
    out = E.expert_mlp(x, p["router"], E.quantize_block_weights(p["w_in"]), E.quantize_block_weights(p["w_out"]), 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.float().sum().backward()
    E.check_device_errors()


def test_without_the_new_arguments():
    """The layer as it was: the same bits as its operators called one by one."""
    g = gen(7)
    p = params(g, 200, 64, 96, 4, torch.bfloat16, False)
    out = E.expert_mlp(p["x"], p["router"], p["w_in"], p["w_out"], 2)
    weights, experts = E.route_experts(p["x"].float() @ p["router"], 2)
    plan = E.plan_experts(experts, 4)
    gate, up = E.grouped_matmul(p["x"], p["w_in"], plan, gather=True).chunk(2, 1)
    y = E.grouped_matmul(torch.nn.functional.silu(gate) * up, p["w_out"], plan)
    assert torch.equal(out, E.combine_experts(y, weights, plan))


def test_captured_training_step():
    """A step of the whole block captured twice, and replayed on new tokens. (No eager graph of the leaves may live
    meanwhile: torch then refuses any capture of a backward pass.)"""
    g = gen(9)
    p = params(g, 260, 128, 96, 4, torch.bfloat16, True)
    dout = randn(g, 260, 128, dtype=torch.bfloat16)
    for t in p.values():
        t.requires_grad_()

    def step():
        out = call(p, 2, "gelu_tanh", 0.5)
        return (out.detach(), *torch.autograd.grad(out, list(p.values()), dout))

    step()
    graphs, kept = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(step())
        graphs.append(graph)
    new = randn(g, 260, 128, dtype=torch.bfloat16)
    with torch.no_grad():
        p["x"].copy_(new)
    want = step()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in kept:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    E.check_device_errors()


def test_refusals():
    g = gen(1)
    p = params(g, 20, 64, 32, 4, torch.bfloat16, False)
    i8 = E.quantize_experts(p["w_in"]), E.quantize_experts(p["w_out"])
    f8 = E.quantize_block_weights(p["w_in"]), E.quantize_block_weights(p["w_out"])
    with pytest.raises(ValueError, match="silu"):
        E.expert_mlp(p["x"], p["router"], *i8, 2, activation="gelu")
    with pytest.raises(TypeError):
        E.expert_mlp(p["x"], p["router"], i8[0], f8[1], 2)
    with pytest.raises(ValueError, match="activation"):
        E.expert_mlp(p["x"], p["router"], p["w_in"], p["w_out"], 2, activation="swish")


def test_two_threads_and_streams():
    """Two programs at once, each on a stream of its own: what each gets alone."""
    import threading
    g = gen(21)
    sets = [params(g, T, 192, 160, 6, torch.bfloat16, True) for T in (700, 37)]
    weights = [(E.quantize_block_weights(p["w_in"]), E.quantize_block_weights(p["w_out"])) for p in sets]
    douts = [torch.ones_like(p["x"]) for p in sets]
    for p in sets:
        for t in p.values():
            t.requires_grad_()

    def step(i):
        p = sets[i]
        out = call(p, 2, "silu", 0.5)
        grads = torch.autograd.grad(out, list(p.values()), douts[i])
        with torch.no_grad():
            served = E.expert_mlp(p["x"], p["router"], *weights[i], 3, norm_in=p["norm_in"], gate=p["gate"])
        return (out.detach(), served, *grads)

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def program(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[i].append(step(i))
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=program, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in (0, 1):
        assert len(got[i]) == 8
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))
    E.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_tensor_in_two_places(dtype):
    """The stream itself as a block's output, one weight for both norms, and the gate: the gradients add up as those
    of tensors of their own do."""
    g = gen(23)
    x, w = randn(g, 90, 136, dtype=dtype), (1 + randn(g, 136, scale=0.2)).to(dtype)
    dout, dy = randn(g, 90, 136, dtype=dtype), randn(g, 90, 136, dtype=dtype)
    apart = [t.clone().requires_grad_() for t in (x, x, w, w, x)]
    out, y = E.residual_norm(*apart, scale=0.25)
    d = torch.autograd.grad((out, y), apart, (dout, dy))
    x.requires_grad_()
    w.requires_grad_()
    out2, y2 = E.residual_norm(x, x, w, w, x, scale=0.25)
    dx, dw = torch.autograd.grad((out2, y2), (x, w), (dout, dy))
    assert torch.equal(out, out2) and torch.equal(y, y2)
    # two sums in the tensors' type, in whatever order: each is off by half a step of its result at most
    size = d[0].double().abs() + d[1].double().abs() + d[4].double().abs()
    unit = torch.finfo(dtype).eps / 2
    assert bool(((dx.double() - (d[0].double() + d[1].double() + d[4].double())).abs() <= 2.01 * unit * size).all())
    both = d[2].double() + d[3].double()
    assert bool(((dw.double() - both).abs() <= 1.01 * unit * both.abs()).all())


def routed_ref(p, experts, act, scale, eps):
    """The block in 64 bits for a routing that is given, differentiable."""
    x = p["x"]
    n = rms(x, p["norm_in"], eps)
    weights = torch.softmax((n @ p["router"]).gather(1, experts), 1)
    y = torch.zeros_like(x)
    F = p["w_out"].shape[1]
    for e in range(p["w_in"].shape[0]):
        for j in range(experts.shape[1]):
            at = (experts[:, j] == e).nonzero()[:, 0]
            h = n[at] @ p["w_in"][e]
            y = y.index_add(0, at, weights[at, j, None] * ((_Act.apply(h[:, :F], act) * h[:, F:]) @ p["w_out"][e]))
    return x + scale * p["gate"] * rms(y, p["norm_out"], eps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_training_16_bits_as_routed(dtype, act):
    """Gradients of a step against the formulas' for the routing that the layer itself took, so that what is left are
    roundings: of the normalised input, the hidden rows, the experts' rows, their sum and the result, and backwards of
    the same and of the hidden rows' two halves. Each is at most a unit of its values, in the norm a unit over the square
    root of three; a dozen in a chain, were all of them alike, are 12 / sqrt(3) = 7 units. relu's derivative jumps: the
    normalised input's rounding moves a gate of spread s by d, 0.8 s u / sqrt(3) in the mean, and one in d / (s sqrt(2 pi))
    = 0.18 u of them changes sides of zero, 0.37 u of the half that counts; whole values come or go, so in the norm of the
    gate's gradient sqrt(0.37 u), whatever else is exact."""
    g = gen(len(act))
    p = params(g, 700, 128, 192, 4, dtype, True)
    for t in p.values():
        t.requires_grad_()
    out = call(p, 2, act, 0.5)
    dout = randn(g, 700, 128, dtype=dtype)
    got = torch.autograd.grad(out, list(p.values()), dout)
    with torch.no_grad():
        experts = E.route_experts(E.rms_norm(p["x"], p["norm_in"]).float() @ p["router"].float(), 2)[1].long()
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    ref = routed_ref(q, experts, act, 0.5, 1e-6)
    want = torch.autograd.grad(ref, list(q.values()), dout.double())
    unit = torch.finfo(dtype).eps / 2
    for name, a, b in zip(("out", *p), (out.detach(), *got), (ref.detach(), *want)):
        off = float((a.double() - b).norm() / b.norm())
        assert off <= 8 * unit + (math.sqrt(0.37 * unit) if act == "relu" else 0.0), (name, off / unit)
