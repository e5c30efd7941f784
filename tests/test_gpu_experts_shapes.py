"""Grouped products on every tile shape, each with ragged groups, several tiles a CTA, even and odd channels.

The shapes of long groups are reached by wide products of little depth (or, in
the gradients, the reverse), so that the 64-bit reference stays quick. Every
case names the kernel that it is for. Bounds as in ``test_gpu_experts``."""

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L
from test_gpu_experts import TYPES, check_int8, gen, grouped_ref, int8_ref, int8s, make_plan, near, randn

pytestmark = pytest.mark.gpu

DEV = "cuda"
CODE = {torch.float32: L.ES_F32, torch.bfloat16: L.ES_BF16, torch.float16: L.ES_F16}
LONG = [200, 701, 256, 0, 513, 390, 640, 511, 257]          # a mean past 240 rows
SHORT = [10 + 37 * i % 91 for i in range(58)] + [0, 129]   # 10 to 100 rows, none, and a tile and one
FEW = [i % 9 for i in range(80)] + [65]                    # up to 8 rows, and a tile and one


def path_of(dtype, plan, K, N):
    return L.lib().es_grouped_matmul_path(CODE[dtype], plan.num_experts, K, N, plan.num_rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,wide,path", [(LONG, 4104, L.ES_GROUPED_WIDE), (LONG, 4101, L.ES_GROUPED_WIDE),
                                             (SHORT, 1032, L.ES_GROUPED_MIDDLE), (SHORT, 1029, L.ES_GROUPED_MIDDLE),
                                             (FEW, 1032, L.ES_GROUPED_NARROW), (FEW, 1029, L.ES_GROUPED_NARROW)])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_shapes(dtype, sizes, wide, path, backward, transposed, gather):
    """Forward from a little depth to many channels, or (backward) the rows' gradient the same way."""
    k = 2 if gather and sum(sizes) % 2 == 0 else 1
    plan = make_plan(sizes, k, dropped=4 * k)
    K, N = (wide, 136) if backward else (136, wide)
    if dtype == torch.float32:  # Middle's part is Wide's and the few rows' kernel's
        path = {L.ES_GROUPED_MIDDLE: L.ES_GROUPED_WIDE}.get(path, path)
        if path == L.ES_GROUPED_NARROW and wide % 4 == 0:
            path = L.ES_GROUPED_FEW
    assert path_of(dtype, plan, N if backward else K, K if backward else N) == path
    g = gen(wide + len(sizes))
    x = randn(g, plan.num_tokens if gather else plan.num_rows, K, dtype=dtype).requires_grad_()
    w = randn(g, len(sizes), *((N, K) if transposed else (K, N)), dtype=dtype, scale=K ** -0.5)
    w = (w.transpose(1, 2) if transposed else w).requires_grad_()
    dy = randn(g, plan.num_rows, N, dtype=dtype)
    y = E.grouped_matmul(x, w, plan, gather=gather)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ry, my, rx, mx, rw, mw = grouped_ref(x, w, plan, gather, dy)
    near(y.detach(), ry, my, K, dtype)
    near(dx, rx, mx, N + k, dtype)
    near(dw, rw, mw, max(sizes), dtype)
    kept = sum(sizes)
    assert not y[kept:].any()
    E.check_device_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,N,path", [(LONG, 4104, L.ES_GROUPED_WIDE), (LONG, 4101, L.ES_GROUPED_WIDE),
                                          (SHORT, 1032, L.ES_GROUPED_MIDDLE), (SHORT, 1029, L.ES_GROUPED_MIDDLE),
                                          (FEW, 1032, L.ES_GROUPED_NARROW), (FEW, 1029, L.ES_GROUPED_NARROW),
                                          ([3, 0, 60, 5], 264, L.ES_GROUPED_SPLIT)])
@pytest.mark.parametrize("K", [144, 2053])
@pytest.mark.parametrize("gather", [False, True])
def test_int8_shapes(dtype, sizes, N, path, K, gather):
    k = 2 if gather and sum(sizes) % 2 == 0 else 1
    plan = make_plan(sizes, k, dropped=4 * k)
    if path == L.ES_GROUPED_SPLIT and K < 1024:
        path = L.ES_GROUPED_NARROW
    assert L.lib().es_int8_matmul_path(plan.num_experts, K, N, plan.num_rows) == path
    g = gen(K + N)
    q, wq = int8s(g, plan.num_tokens if gather else plan.num_rows, K), int8s(g, len(sizes), N, K)
    s = torch.rand(q.shape[0], generator=g, device=DEV) * 2.0 ** -12
    ws = torch.rand(len(sizes), N, generator=g, device=DEV)
    y = E.int8_matmul(q, s, wq, ws, plan, gather=gather, out_dtype=dtype)
    check_int8(y, int8_ref(q, s, wq, ws, plan, gather), dtype)
    E.check_device_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,N,path", [(2501, 4104, L.ES_GROUPED_WIDE), (2500, 4101, L.ES_GROUPED_WIDE),
                                         (235, 19208, L.ES_GROUPED_MIDDLE), (235, 19203, L.ES_GROUPED_MIDDLE),
                                         (7, 12293, L.ES_GROUPED_NARROW), (70, 4104, L.ES_GROUPED_SPLIT)])
def test_int8_dense_shapes(dtype, rows, N, path):
    K = 1040
    assert L.lib().es_int8_matmul_path(0, K, N, rows) == path
    g = gen(rows)
    q, wq = int8s(g, rows, K), int8s(g, N, K)
    s, ws = torch.rand(rows, generator=g, device=DEV) * 2.0 ** -12, torch.rand(N, generator=g, device=DEV)
    check_int8(E.int8_matmul(q, s, wq, ws, out_dtype=dtype), int8_ref(q, s, wq, ws, None, False), dtype)
