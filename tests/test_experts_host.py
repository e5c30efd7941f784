"""Expert operators: what is decided on the host, before any launch (no GPU needed)."""

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L

FAKE = 1 << 20  # an aligned address that is never read


def rows_args(K=64, N=128, dtype=L.ES_BF16, x=FAKE, w=FAKE, x_stride=None, order=None, strides=None, experts=4,
              rows=100):
    x_rows = rows if order is None else 50
    se, sk, sn = strides or (K * N, N, 1)
    return (x, dtype, x_rows, x_stride or K, w, experts, K, N, se, sk, sn, FAKE, order, 2, rows)


def test_workspace_sizes():
    lib = L.load()
    size = lib.es_grouped_matmul_workspace_size
    assert size(*rows_args()) == 0                                    # read where it lies
    assert size(*rows_args(order=FAKE)) >= 100 * 64 * 2               # routed rows
    assert size(*rows_args(x=FAKE + 2)) >= 100 * 64 * 2               # an address that TMA cannot read
    assert size(*rows_args(N=101)) >= 4 * 64 * 101 * 2                # a row pitch of no whole 16 bytes
    assert size(*rows_args(strides=(64 * 128, 1, 64))) == 0           # the transposed view
    assert size(*rows_args(strides=(2 * 64 * 128, 256, 2))) >= 4 * 64 * 128 * 2
    assert size(*rows_args(strides=(0, 128, 1))) == 0                 # one matrix for all experts
    assert size(*rows_args(dtype=L.ES_F32)) >= 3 * 2 * (100 * 64 + 4 * 64 * 128)
    assert size(*rows_args(dtype=L.ES_F32, rows=20)) == 0             # few rows: read where they lie
    assert size(*rows_args(dtype=L.ES_F32, rows=20, w=FAKE + 4)) > 0
    assert size(*rows_args(K=0)) == 0 and size(*rows_args(rows=0)) == 0
    plan = lib.es_expert_plan_workspace_size
    assert plan(100, 8) == 0 and plan(1 << 20, 8) > 0 and plan(1 << 20, 1024) > plan(1 << 20, 8)


def test_entry_points_refuse():
    lib = L.load()
    inv, uns, ws = L.ES_ERR_INVALID, L.ES_ERR_UNSUPPORTED, L.ES_ERR_WORKSPACE
    route = lib.es_route_experts
    assert route(FAKE, L.ES_F32, 4, 8, 8, 9, 1, FAKE, FAKE, None) == inv
    assert route(FAKE, L.ES_F32, 4, 8, 8, 0, 1, FAKE, FAKE, None) == inv
    assert route(FAKE, L.ES_F32, 4, 2000, 2000, 2, 1, FAKE, FAKE, None) == uns
    assert route(FAKE, L.ES_F32, 4, 64, 64, 33, 1, FAKE, FAKE, None) == uns
    assert route(FAKE, L.ES_F64, 4, 8, 8, 2, 1, FAKE, FAKE, None) == uns
    assert route(None, L.ES_F32, 4, 8, 8, 2, 1, FAKE, FAKE, None) == inv
    assert route(None, L.ES_F32, 0, 8, 8, 2, 1, None, None, None) == L.ES_OK
    assert lib.es_expert_plan(FAKE, 1 << 20, 8, None, 0, FAKE, FAKE, FAKE, None, None) == ws
    assert lib.es_expert_plan(FAKE, 10, 0, None, 0, FAKE, FAKE, FAKE, None, None) == inv
    assert lib.es_expert_plan(FAKE, 10, 1025, None, 0, FAKE, FAKE, FAKE, None, None) == uns
    rows = lib.es_grouped_matmul
    assert rows(*rows_args(order=FAKE), FAKE, L.ES_BF16, None, 0, None, None) == ws
    assert rows(*rows_args(), FAKE, L.ES_F16, None, 0, None, None) == uns      # neither x's type nor fp32
    assert rows(*rows_args(), None, L.ES_BF16, None, 0, None, None) == inv
    assert rows(*rows_args(dtype=L.ES_F64), FAKE, L.ES_F64, None, 0, None, None) == uns
    assert rows(*rows_args(experts=0), FAKE, L.ES_BF16, None, 0, None, None) == inv
    assert rows(*rows_args(rows=-1), FAKE, L.ES_BF16, None, 0, None, None) == inv
    assert rows(*rows_args(rows=0), None, L.ES_BF16, None, 0, None, None) == L.ES_OK
    int8 = (FAKE, FAKE, 10, 64, FAKE, FAKE, 0, 64, 128, 0, 64, None, None, 1, 10)
    assert lib.es_int8_matmul(*int8, FAKE, L.ES_F64, None, 0, None, None) == uns
    deep = (FAKE, FAKE, 10, 200000, FAKE, FAKE, 0, 200000, 128, 0, 200000, None, None, 1, 10)
    assert lib.es_int8_matmul(*deep, FAKE, L.ES_BF16, None, 0, None, None) == uns
    assert lib.es_combine_experts(FAKE, L.ES_BF16, 10, 64, None, FAKE, 5, 2, 64, FAKE, L.ES_F16, None) == uns
    assert lib.es_quantize_rows(FAKE, L.ES_F64, 4, 64, 64, FAKE, FAKE, None) == uns


def test_cpu_tensors_are_refused():
    x, e = torch.ones(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: E.route_experts(x, 2), lambda: E.plan_experts(e, 8), lambda: E.quantize_rows(x),
                 lambda: E.ExpertPlan(e[0], e[0], e[:1]),
                 lambda: E.int8_matmul(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: E.grouped_matmul(x, x[None], None), lambda: E.combine_experts(x, x, None),
                 lambda: E.route_experts([[1.0]], 1)):
        with pytest.raises(TypeError):
            call()
