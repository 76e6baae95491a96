"""The streamed forms of rr_unpermute_norm and its backward pass with parts left
out: no post_gamma, gate or pre_gamma, no d_residual_out or d_normed, skipped
routes, in place. Bounds as in test_gpu_unpermute_norm."""
from __future__ import annotations

import pytest
import torch

from test_gpu_unpermute_norm import BF16, EPS, FP32, Inputs, check_backward, check_forward

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


# Enough tokens for the streamed gradient in each of its widths: one warp and
# several per token, two routes or more, rows that start anywhere.
GRADIENT = [(600, 2, 512), (1201, 5, 250), (300, 2, 4100)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", GRADIENT, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")], ids=str)
def test_gradient_without_norms_of_rows_that_are_not_finite(cuda, shape, dtype, bad):
    """Without norms the gradient of the residual and of the routes' rows is
    linear in d_residual_out, whatever the forward values are; a weight's gradient
    depends on its own route's row only."""
    t, k, n = shape
    i = Inputs(*shape, dtype, cuda, 5, post=False, pre=False)
    clean = i.backward(None)
    i.res[7, n // 2] = bad
    i.res[t - 1] = bad
    row = int(i.pos[11, 0])
    i.yp[row, 3] = bad
    got = i.backward(None)
    assert torch.equal(got["d_residual"], clean["d_residual"])
    assert torch.equal(got["d_yp"], clean["d_yp"])
    want = clean["d_w"].clone()
    assert not torch.isfinite(got["d_w"][11, 0])
    want[11, 0] = got["d_w"][11, 0] = 0.0
    assert torch.equal(got["d_w"], want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", GRADIENT, ids=str)
def test_gradient_without_the_last_norm_of_a_residual_that_is_not_finite(cuda, shape, dtype):
    """Without a gradient through the last norm the residual's values take no part."""
    i = Inputs(*shape, dtype, cuda, 6, pre=False)
    c = (i.yp.double()[i.pos.long()] * i.w.double()[..., None]).sum(1)
    inv = torch.ones(shape[0], 2, device=cuda)
    inv[:, 0] = torch.rsqrt((c * c).mean(1) + EPS).float()
    clean = i.backward(inv)
    i.res[3], i.res[8, 1] = float("inf"), float("nan")
    got = i.backward(inv)
    for name, t in clean.items():
        if t is not None:
            assert torch.equal(got[name], t), name


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(1650, 2, 1027), (8003, 3, 333), (21000, 1, 131)], ids=str)
def test_the_last_row_comes_first(cuda, shape, dtype):
    """The buffer's last row, whose end is copied by element, among the first tokens:
    later rows are copied into the same place whole."""
    i = Inputs(*shape, dtype, cuda, 71)
    flat = i.pos.view(-1)
    for token in (0, 1, 5):
        last = int((flat == flat.numel() - 1).nonzero()[0, 0])
        to = token * shape[1]
        flat[last], flat[to] = flat[to].item(), flat[last].item()
        out, normed, inv = i.forward()
        check_forward(i, out, normed, dtype)
        check_backward(i, i.backward(inv), dtype)
