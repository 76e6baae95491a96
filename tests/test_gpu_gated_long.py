"""Contractions that take the tensor-core engine seconds: no wait gives up before
a tile's products are done."""
from __future__ import annotations

import pytest
import torch

from expert_block_reference import offsets_of
from test_gpu_gated import BF16, no_device_error

import raggedroute_b200 as rr

pytestmark = pytest.mark.gpu


def test_a_contraction_of_seconds(cuda):
    """K = 2^30, the largest (one tile of 16.8 million k-blocks), zero but for its ends and
    middle: every sum is exact."""
    k, n, rows = 2 ** 30, 8, 5
    at = torch.tensor([0, 1, k // 2 + 3, k - 1], device=cuda)
    x = torch.zeros(rows, k, dtype=BF16, device=cuda)
    wg, wu = (torch.zeros(1, k, n, dtype=BF16, device=cuda) for _ in range(2))
    x[:, at] = torch.tensor([1.0, 2.0, 4.0, 8.0], dtype=BF16, device=cuda)
    wg[0, at] = torch.arange(1.0, n + 1, device=cuda).to(BF16)
    wu[0, at] = -2.0
    h = torch.empty(rows, n, dtype=BF16, device=cuda)
    gu = torch.empty(rows, 2 * n, device=cuda)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    rr.grouped_gated_gemm(x, wg, wu, offsets_of([rows], cuda), h, gate_up=gu, activation="relu")
    end.record()
    no_device_error()
    end.synchronize()
    assert start.elapsed_time(end) > 2000  # the limit of a wait on anything shorter
    g = 15 * torch.arange(1.0, n + 1, device=cuda)
    assert torch.equal(gu, torch.cat((g, torch.full_like(g, -30.0))).expand(rows, -1))
    assert torch.equal(h, (g * -30.0).to(BF16).expand(rows, -1))
    del x, wg, wu
    torch.cuda.empty_cache()  # 45 GB
