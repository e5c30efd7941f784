"""Gated products, 8-bit floating point and norms: what is decided on the host, before any launch (no GPU needed)."""

import pytest
import torch

import einjax_b200 as E
from einjax_b200 import _lib as L

FAKE = 1 << 20  # an aligned address that is never read
F32, BF16, F16, F64 = L.ES_F32, L.ES_BF16, L.ES_F16, L.ES_F64
OK, INV, UNS, WS = L.ES_OK, L.ES_ERR_INVALID, L.ES_ERR_UNSUPPORTED, L.ES_ERR_WORKSPACE


def gated_args(K=64, F=128, dtype=BF16, x=FAKE, w=FAKE, order=None, strides=None, experts=4, rows=100, offsets=FAKE):
    se, sk, sn = strides or (2 * K * F, 2 * F, 1)
    return (x, dtype, 50 if order else rows, K, w, experts, K, F, se, sk, sn, offsets, order, 2, rows)


def test_gated_workspace():
    size = L.load().es_gated_matmul_workspace_size
    assert size(*gated_args()) == 0                                   # read where it lies
    assert size(*gated_args(order=FAKE)) >= 100 * 64 * 2              # routed rows
    assert size(*gated_args(F=101)) >= 4 * 64 * 2 * 101 * 2           # up starts at no whole 16 bytes
    assert 0 < size(*gated_args(F=132)) < 2 * 4 * 64 * 136 * 2        # gate is read where it lies, up is copied
    assert size(*gated_args(strides=(2 * 64 * 128, 1, 64))) == 0      # the transposed view
    assert size(*gated_args(dtype=F32)) >= 100 * 256 * 4              # the product in fp32
    assert size(*gated_args(K=20000, dtype=F16)) >= 100 * 256 * 4
    assert size(*gated_args(experts=0, offsets=None)) == 0
    assert size(*gated_args(rows=0)) == 0 and size(*gated_args(F=0)) == 0


def test_gated_refuses():
    lib = L.load()
    call = lib.es_gated_matmul
    tail = (FAKE, None, None, 0, None, None)
    assert call(*gated_args(), 4, *tail) == INV and call(*gated_args(), -1, *tail) == INV
    assert call(*gated_args(order=FAKE), 0, *tail) == WS
    assert call(*gated_args(dtype=F32), 0, *tail) == WS
    assert call(*gated_args(dtype=F64), 0, FAKE, None, FAKE, 1 << 30, None, None) == UNS
    assert call(*gated_args(), 0, None, None, None, 0, None, None) == INV
    assert call(*gated_args(experts=0), 0, *tail) == INV              # offsets without groups
    assert call(*gated_args(experts=1025), 0, FAKE, None, FAKE, 1 << 30, None, None) == UNS
    assert call(*gated_args(rows=-1), 0, *tail) == INV
    assert call(*gated_args(rows=0), 0, None, None, None, 0, None, None) == OK
    grad = lib.es_gated_matmul_grad
    assert grad(None, BF16, 8, FAKE, 4, 8, None, FAKE, None) == INV
    assert grad(FAKE, F64, 8, FAKE, 4, 8, None, FAKE, None) == UNS
    assert grad(None, BF16, 8, None, 0, 8, None, None, None) == OK


@pytest.mark.parametrize("dtype,experts,K,F,rows,path", [
    # by the mean of the rows a group, where the tiles then fill the SMs (lanes are h's channels)
    (BF16, 60, 2048, 1408, 60, L.ES_GROUPED_MIDDLE), (BF16, 60, 2048, 1408, 60 * 112, L.ES_GROUPED_MIDDLE),
    (BF16, 60, 2048, 1408, 60 * 113, L.ES_GROUPED_WIDE), (BF16, 80, 136, 128, 400, L.ES_GROUPED_NARROW),
    (F16, 0, 4096, 8192, 8192, L.ES_GROUPED_WIDE), (BF16, 0, 4096, 2048, 16, L.ES_GROUPED_SPLIT),
    (BF16, 0, 128, 2048, 16, L.ES_GROUPED_NARROW),
    # one chain of sums in one kernel; fp32 and longer sums in two
    (F16, 0, 16384, 8192, 8192, L.ES_GROUPED_WIDE), (F16, 0, 16385, 8192, 8192, L.ES_GATED_TWO),
    (BF16, 0, 65536, 1024, 4096, L.ES_GROUPED_MIDDLE), (BF16, 0, 65537, 1024, 4096, L.ES_GATED_TWO),
    (F32, 8, 64, 64, 64, L.ES_GATED_TWO),
    (F64, 8, 64, 64, 64, -1), (BF16, 1025, 64, 64, 64, -1), (BF16, 8, 0, 64, 64, -1), (BF16, 8, 64, 64, 0, -1),
])
def test_gated_path(dtype, experts, K, F, rows, path):
    assert L.load().es_gated_matmul_path(dtype, experts, K, F, rows) == path


@pytest.mark.parametrize("experts,K,N,rows,path", [
    (0, 4096, 4096, 16, L.ES_GROUPED_SPLIT), (0, 4096, 8192, 8191, L.ES_GROUPED_WIDE),
    (64, 2048, 2816, 64 * 128, L.ES_GROUPED_NARROW), (64, 2048, 2816, 64 * 129, L.ES_GROUPED_WIDE),
    (0, 256, 4096, 16, L.ES_GROUPED_NARROW), (0, 64, 0, 64, -1), (1025, 64, 64, 64, -1), (-1, 64, 64, 64, -1),
])
def test_fp8_path(experts, K, N, rows, path):
    assert L.load().es_fp8_matmul_path(experts, K, N, rows) == path


def fp8_args(K=256, N=128, q=FAKE, w=FAKE, x_stride=None, n_stride=None, order=None, experts=4, rows=100, offsets=FAKE):
    return (q, FAKE, 50 if order else rows, x_stride or K, w, FAKE, experts, K, N, (n_stride or K) * N, n_stride or K,
            offsets, order, 2, rows)


def test_fp8_host():
    lib = L.load()
    size, call = lib.es_fp8_matmul_workspace_size, lib.es_fp8_matmul
    assert size(*fp8_args()) == 0 and size(*fp8_args(order=FAKE)) >= 100 * 256
    assert size(*fp8_args(K=100)) >= 100 * 100 + 4 * 128 * 100       # a row pitch of no whole 16 bytes
    assert size(*fp8_args(q=FAKE + 1)) >= 100 * 256 and size(*fp8_args(w=FAKE + 8)) >= 4 * 128 * 256
    tail = (FAKE, BF16, None, 0, None, None)
    assert call(*fp8_args(order=FAKE), *tail) == WS
    assert call(*fp8_args(), FAKE, F64, None, 0, None, None) == UNS
    assert call(*fp8_args(), None, BF16, None, 0, None, None) == INV
    assert call(*fp8_args(q=None), *tail) == INV and call(*fp8_args(experts=0), *tail) == INV
    assert call(*fp8_args(rows=0), None, BF16, None, 0, None, None) == OK
    quant = lib.es_quantize_blocks
    assert quant(FAKE, F64, 4, 64, 64, -1, FAKE, FAKE, None) == UNS
    assert quant(FAKE, BF16, 4, 64, 64, 4, FAKE, FAKE, None) == INV
    assert quant(None, BF16, 4, 64, 64, -1, FAKE, FAKE, None) == INV
    assert quant(None, BF16, 0, 64, 64, -1, None, None, None) == OK
    assert lib.es_quantize_block_weights(FAKE, F64, 1, 8, 8, FAKE, FAKE, None) == UNS
    assert lib.es_quantize_block_weights(FAKE, BF16, 1 << 20, 1 << 20, 1 << 20, FAKE, FAKE, None) == UNS
    assert lib.es_quantize_block_weights(None, BF16, 0, 8, 8, None, None, None) == OK


def norm(**kw):
    a = dict(x=FAKE, xs=64, h=FAKE, hs=64, dtype=BF16, rows=4, width=64, norm_in=FAKE, norm_out=FAKE, wd=BF16, gate=None,
             kind=L.ES_GATE_NONE, gs=0, out=FAKE, y=FAKE)
    a.update(kw)
    return L.load().es_residual_norm(a["x"], a["xs"], a["h"], a["hs"], a["dtype"], a["rows"], a["width"], a["norm_in"],
                                     a["norm_out"], a["wd"], a["gate"], a["kind"], a["gs"], 1.0, 1e-6, a["out"], a["y"],
                                     None, None)


def test_norm_refuses():
    assert norm(dtype=F64) == UNS and norm(wd=F16) == UNS
    assert norm(x=None) == INV and norm(y=None) == INV and norm(out=None) == INV
    assert norm(gate=FAKE) == INV and norm(kind=L.ES_GATE_TOKEN) == INV and norm(gate=FAKE, kind=7) == INV
    assert norm(h=None) == INV and norm(h=None, norm_out=None, norm_in=None) == INV
    assert norm(rows=-1) == INV
    assert norm(rows=0, x=None, h=None, out=None, y=None) == OK and norm(width=0, norm_in=None, norm_out=None) == OK
    size = L.load().es_residual_norm_grad_workspace_size
    for dtype in (F32, BF16):
        for width in (1, 5, 8, 100, 4096, 5001, 16384, 100000):  # every width has a form, short ones too
            assert size(dtype, 1, width, 1) >= 4 * width
            assert size(dtype, 1 << 20, width, 3) >= 3 * size(dtype, 1, width, 1)
    assert size(BF16, 0, 64, 3) == 0 and size(BF16, 64, 64, 0) == 0


def test_cpu_tensors_are_refused():
    x, w = torch.ones(4, 8), torch.ones(8)
    f8 = torch.ones(4, 8).to(torch.float8_e4m3fn)
    for call in (lambda: E.rms_norm(x, w), lambda: E.residual_norm(x, x), lambda: E.gated_matmul(x, x.t()),
                 lambda: E.quantize_blocks(x), lambda: E.quantize_block_weights(x), lambda: E.fp8_matmul(f8, x, f8, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: E.rms_norm([1.0], w), lambda: E.gated_matmul(None, x), lambda: E.quantize_blocks(None),
                 lambda: E.fp8_matmul(None, x, f8, x)):
        with pytest.raises(TypeError):
            call()
