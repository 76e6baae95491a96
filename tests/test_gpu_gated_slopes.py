"""The activations' slopes in rr_grouped_gated_gemm_backward far out."""
from __future__ import annotations

import pytest
import torch

from expert_block_reference import offsets_of
from test_gpu_gated import BF16, FP32, backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [3, 64])
def test_gelu_slope_far_out(cuda, rows, dtype):
    """gelu_tanh is g or 0 from a few tens on, and its slope 1 or 0, as far as
    floats reach (powers of two: every sum here is exact)."""
    far = [2.0 ** e * s for e in (5, 62, 64, 66, 100, 126) for s in (1, -1)] + [64.0, -64.0] * 2
    g = torch.tensor(far, device=cuda)
    x = torch.ones(rows, 8, dtype=dtype, device=cuda)
    wg = torch.ones(1, 8, 16, dtype=dtype, device=cuda)
    dh = torch.full((rows, 16), 2.0 ** -10, dtype=dtype, device=cuda)
    gu = torch.cat((g, torch.ones_like(g))).expand(rows, 32).contiguous()
    dx, dwg, dwu = backward(x, wg, torch.zeros_like(wg), offsets_of([rows], cuda), gu, dh,
                            "gelu_tanh")
    slope = (g > 0).double() * 2.0 ** -10
    assert torch.equal(dwg[0].double(), (rows * slope).expand(8, 16))
    assert torch.equal(dwu[0].double(), (rows * slope * g.double()).expand(8, 16))
    assert torch.equal(dx.double(), slope.sum().expand(rows, 8))
