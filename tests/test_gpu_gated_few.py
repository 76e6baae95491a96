"""rr_grouped_gated_gemm for a few rows, where a cluster's blocks share the
contraction and their partial sums meet in the first one. Bounds as in
test_gpu_gated."""
from __future__ import annotations

import math

import pytest
import torch

from expert_block_reference import gated, normwise
from test_gpu_gated import BF16, FP32, forward, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("counts", [[1], [0, 2], [4], [1, 0, 3]], ids=str)
@pytest.mark.parametrize("k,n", [(8192, 64), (4099, 130), (600, 40), (64, 2048)])
def test_partial_sums_of_a_cluster(cuda, counts, k, n, dtype):
    x, wg, wu, off, _ = make(counts, 0, k, n, dtype, cuda, seed=7)
    h, gu = forward(x, wg, wu, off)
    g, u, want = gated(x, wg, wu, off)
    assert normwise(gu, torch.cat((g, u), 1)) < 2.0 ** -19
    assert normwise(h, want) < (2.0 ** -8 / math.sqrt(3) if dtype == BF16 else 2.0 ** -19)
    for _ in range(20):
        again = forward(x, wg, wu, off)
        assert torch.equal(h, again[0]) and torch.equal(gu, again[1])
