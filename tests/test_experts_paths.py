"""Which kernel a rows' product takes, by its sizes (decided on the host, no GPU needed).

``test_gpu_experts_shapes`` runs every one of them; these pin the rule's two sides."""

import pytest

from einjax_b200 import _lib as L

F32, BF16, F16 = L.ES_F32, L.ES_BF16, L.ES_F16


@pytest.mark.parametrize("dtype,experts,K,N,rows,path", [
    # 16 bits: by the mean of the rows a group, where the tiles fill the SMs
    (BF16, 60, 2048, 2816, 60 * 8, L.ES_GROUPED_NARROW),
    (BF16, 60, 2048, 2816, 60 * 9, L.ES_GROUPED_MIDDLE),
    (BF16, 60, 2048, 2816, 60 * 160, L.ES_GROUPED_MIDDLE),
    (BF16, 60, 2048, 2816, 60 * 161, L.ES_GROUPED_WIDE),
    (F16, 8, 4096, 8192, 16384, L.ES_GROUPED_WIDE),
    # few tiles: Wide wants 74, Middle 148, and a cluster shares the depth of what is less
    (BF16, 1, 4096, 512 * 24, 512, L.ES_GROUPED_MIDDLE),
    (BF16, 1, 4096, 512 * 25, 512, L.ES_GROUPED_WIDE),
    (BF16, 1, 4096, 4096, 16, L.ES_GROUPED_SPLIT),
    (BF16, 4, 256, 4096, 8, L.ES_GROUPED_NARROW),
    (BF16, 1, 128, 4096, 16, L.ES_GROUPED_NARROW),
    # long sums
    (F16, 8, 16384, 8192, 16384, L.ES_GROUPED_WIDE),
    (F16, 8, 16385, 8192, 16384, L.ES_GROUPED_DEEP_WIDE),
    (F16, 60, 16385, 2816, 600, L.ES_GROUPED_DEEP_NARROW),
    (F16, 1, 16385, 4096, 16, L.ES_GROUPED_SPLIT),
    (BF16, 8, 65536, 8192, 16384, L.ES_GROUPED_WIDE),
    (BF16, 8, 65537, 8192, 16384, L.ES_GROUPED_DEEP_WIDE),
    # fp32
    (F32, 36, 2520, 1456, 36 * 24, L.ES_GROUPED_FEW),
    (F32, 36, 2520, 1456, 36 * 24 + 1, L.ES_GROUPED_WIDE),
    (F32, 36, 2520, 1457, 36 * 8, L.ES_GROUPED_NARROW),
    (F32, 36, 2520, 1457, 36 * 9, L.ES_GROUPED_WIDE),
    (F32, 1, 2048, 131, 25, L.ES_GROUPED_SPLIT),
    (F32, 16, 1000, 2024, 3000, L.ES_GROUPED_WIDE),
    (F32, 1, 1 << 20, 4096, 4096, L.ES_GROUPED_WIDE),
    # none
    (L.ES_F64, 8, 64, 64, 64, -1), (BF16, 0, 64, 64, 64, -1), (BF16, 1025, 64, 64, 64, -1), (BF16, 8, 0, 64, 64, -1),
    (BF16, 8, 64, 64, 0, -1),
])
def test_grouped_path(dtype, experts, K, N, rows, path):
    assert L.load().es_grouped_matmul_path(dtype, experts, K, N, rows) == path


@pytest.mark.parametrize("experts,K,N,rows,path", [
    (0, 4096, 4096, 16, L.ES_GROUPED_SPLIT),
    (0, 4096, 8192, 8191, L.ES_GROUPED_WIDE),
    (64, 2048, 1408, 64 * 8, L.ES_GROUPED_NARROW),
    (64, 2048, 1408, 64 * 9, L.ES_GROUPED_MIDDLE),
    (64, 2048, 1408, 64 * 240, L.ES_GROUPED_MIDDLE),
    (64, 2048, 1408, 64 * 241, L.ES_GROUPED_WIDE),
    (8, 131071, 8192, 16384, L.ES_GROUPED_WIDE),
    (8, 131072, 8192, 16384, -1), (0, 64, 0, 64, -1), (1025, 64, 64, 64, -1),
])
def test_int8_path(experts, K, N, rows, path):
    assert L.load().es_int8_matmul_path(experts, K, N, rows) == path
