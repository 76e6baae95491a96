"""The streamed forms of rr_unpermute_norm and its backward pass with parts left
out: no post_gamma, gate or pre_gamma, no d_residual_out or d_normed, skipped
routes, in place. Bounds as in test_gpu_unpermute_norm."""
from __future__ import annotations

import pytest
import torch

from test_gpu_unpermute_norm import BF16, FP32, Inputs, check_forward

pytestmark = pytest.mark.gpu

# (post, gate, pre): all but the whole.
PARTS = [(0, 0, 0), (0, 0, 1), (0, 1, 0), (0, 1, 1), (1, 0, 0), (1, 0, 1), (1, 1, 0)]

# Enough bytes for the streamed forward pass: teams of one warp to sixteen, aligned
# rows and rows that start anywhere, many tokens per team.
FORWARD = [(13201, 2, 512), (3299, 2, 2048), (1701, 2, 4096), (901, 2, 8192), (8003, 3, 333),
           (1650, 2, 1027)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("parts", PARTS, ids=str)
@pytest.mark.parametrize("shape", FORWARD, ids=str)
def test_forward(cuda, shape, parts, dtype):
    """One, two or no sums per token: warps of a team that run ahead do not touch
    what the others still read, so results are right and repeat."""
    post, gate, pre = map(bool, parts)
    i = Inputs(*shape, dtype, cuda, 61, post=post, gate=gate, pre=pre, skip=True)
    out, normed, inv = i.forward()
    check_forward(i, out, normed, dtype)
    for _ in range(3):
        out2, normed2, inv2 = i.forward()
        assert torch.equal(out, out2) and torch.equal(inv, inv2)
        assert normed is None or torch.equal(normed, normed2)
    i.res = i.res.clone()
    out2, normed2, inv2 = i.forward(out=i.res)  # in place
    assert torch.equal(out, out2) and torch.equal(inv, inv2)
    assert normed is None or torch.equal(normed, normed2)
