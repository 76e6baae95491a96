"""The streamed forms of rr_unpermute_norm and its backward pass with parts left
out: no post_gamma, gate or pre_gamma, no d_residual_out or d_normed, skipped
routes, in place. Bounds as in test_gpu_unpermute_norm."""
from __future__ import annotations

import pytest
import torch

from expert_block_reference import half_step
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


# Teams of one warp to sixteen, a wide row, two routes or more, rows of whole granules,
# of pairs and of single elements; tokens that end inside a stage.
GRADIENT_PARTS = [(1201, 2, 250), (600, 2, 512), (601, 4, 264), (601, 2, 4096), (599, 2, 4095),
                  (301, 3, 2050), (299, 2, 8192), (1201, 16, 520)]


def inverse(i: Inputs):
    """The forward pass's inv_rms."""
    return i.forward()[2]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("parts", PARTS, ids=str)
@pytest.mark.parametrize("shape", GRADIENT_PARTS, ids=str)
def test_gradient(cuda, shape, parts, dtype):
    post, gate, pre = map(bool, parts)
    i = Inputs(*shape, dtype, cuda, 81, post=post, gate=gate, pre=pre, skip=True)
    inv = inverse(i)
    got = i.backward(inv)
    check_backward(i, got, dtype)
    again = i.backward(inv)
    i.dro = d = i.dro.clone()
    in_place = i.backward(inv, d_residual=d)  # d_residual over d_residual_out
    for name, t in got.items():
        assert t is None or torch.equal(t, again[name]) and torch.equal(t, in_place[name]), name


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("shape", GRADIENT_PARTS, ids=str)
def test_gradients_that_are_not_given(cuda, shape, post, dtype):
    """No d_residual_out, no d_normed, neither: as if they were zero."""
    i = Inputs(*shape, dtype, cuda, 82, post=post, skip=True)
    inv = inverse(i)
    dro, dn = i.dro, i.dn
    for without in ("dro", "dn"):
        i.dro, i.dn = dro, dn
        setattr(i, without, None)
        got = i.backward(inv)
        setattr(i, without, torch.zeros_like(dn))
        check_backward(i, got, dtype)
    i.dro = i.dn = None
    for name, t in i.backward(inv).items():
        if name == "d_yp":
            t = t[t != 7.0]  # rows that no route names
        assert t is None or not t.any(), name


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(300, 1, 200), (300, 1, 512), (300, 1, 511), (300, 1, 4100),
                                   (5, 1, 33)], ids=str)
def test_weight_gradient_of_a_single_route(cuda, shape, dtype):
    """With a norm of c and one route the weight's gradient cancels but for eps:
      d_w = i1 (<v1, y> - m1 <cn, y>),  v1 = gate post dr,  m1 = mean(v1 cn).
    Each value is within u = (64 + top_k) 2^-24 of the magnitudes it is summed from: dr of
    |dro| + i2 (|v| + |rn| m2), m2 of mean |v||rn|; v1, cn and the dot products three
    more times that, so 4 u of the products' magnitudes."""
    i = Inputs(*shape, dtype, cuda, 83)
    inv = inverse(i)
    got = i.backward(inv)["d_w"][:, 0].double()
    yp, w, res, post, gate, pre = (t.detach() for t in i.leaves())
    y = yp[i.pos[:, 0].long()]
    c = w * y
    i1 = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    cn = c * i1
    r = i.scale * res + gate * post * cn
    i2 = 1 / torch.sqrt((r * r).mean(1, keepdim=True) + EPS)
    rn, v = r * i2, i.dn.double() * pre
    dr = i.dro.double() + i2 * (v - rn * (v * rn).mean(1, keepdim=True))
    v1 = gate * post * dr
    m1 = (v1 * cn).mean(1, keepdim=True)
    want = (i1 * ((v1 * y).sum(1, keepdim=True) - m1 * (cn * y).sum(1, keepdim=True)))[:, 0]
    big = (gate * post).abs() * (i.dro.double().abs() + i2 * (
        v.abs() + rn.abs() * (v * rn).abs().mean(1, keepdim=True)))
    big_m1 = (big * cn.abs()).mean(1, keepdim=True)
    size = (i1 * ((big * y.abs()).sum(1, keepdim=True)
                  + big_m1 * (cn * y).abs().sum(1, keepdim=True)))[:, 0]
    assert bool(((got - want).abs() <= 4 * 65 * 2.0 ** -24 * size).all())
    assert float((4 * 65 * 2.0 ** -24 * size).max()) < 0.3


def check_gradient_elementwise(i: Inputs, got, dtype):
    """Every gradient within the first-order bound of FP32 arithmetic. Each value is
    within u = (64 + top_k) 2^-24 of the magnitudes it is summed from, and carries on the
    errors of what it is computed from (d*). Short rows need this: with N = 1 a norm's
    1/rms reaches 1 / sqrt(eps) = 1000 and its gradient cancels all but eps of itself.
    Twice the bound, for terms of second order and the grouping of the sums."""
    yp, w, res, post, gate, pre = (t.detach() for t in i.leaves())
    t, k, n = *i.pos.shape, i.res.shape[1]
    u = (64 + k) * 2.0 ** -24
    there = (i.pos >= 0) & (i.pos < t * k)
    y = yp[i.pos.clamp(0, t * k - 1).long()] * there[..., None]
    w = (w * there)[..., None]

    def mean(v):
        return v.mean(1, keepdim=True)

    c, dc = (w * y).sum(1), u * (w * y).abs().sum(1)
    i1 = 1 / torch.sqrt(mean(c * c) + EPS)
    e1 = i1 * mean(dc * dc).sqrt() + u  # relative, of i1
    cn, dcn = c * i1, i1 * dc + (c * i1).abs() * e1
    f = gate * post
    r = i.scale * res + f * cn
    dr_ = u * (abs(i.scale) * res.abs() + (f * cn).abs()) + f.abs() * dcn
    i2 = 1 / torch.sqrt(mean(r * r) + EPS)
    e2 = i2 * mean(dr_ * dr_).sqrt() + u
    rn, drn = r * i2, i2 * dr_ + (r * i2).abs() * e2
    dro, dn = i.dro.double(), i.dn.double()
    v = dn * pre
    m2, dm2 = mean(v * rn), mean(v.abs() * (drn + u * rn.abs()))
    x, big_x = v - rn * m2, v.abs() + (rn * m2).abs()
    dr = dro + i2 * x
    ddr = u * dro.abs() + i2 * ((u + e2) * big_x + drn * m2.abs() + rn.abs() * dm2)
    v1, dv1 = f * dr, f.abs() * (ddr + u * (dro.abs() + i2 * big_x))
    big_cn = i1 * (w * y).abs().sum(1)
    m1 = mean(v1 * cn)
    dm1 = mean(dv1 * big_cn + v1.abs() * (dcn + u * big_cn))
    dct = i1 * (v1 - cn * m1)
    ddct = i1 * ((u + e1) * (v1.abs() + (cn * m1).abs()) + dv1 + dcn * m1.abs() + cn.abs() * dm1)
    half = half_step(dtype)
    named = torch.zeros(t * k, dtype=torch.bool, device=yp.device)
    named[i.pos[there].long()] = True
    want_y, err_y = torch.zeros_like(yp), torch.zeros_like(yp)
    want_y[i.pos[there].long()] = (w * dct[:, None])[there]
    err_y[i.pos[there].long()] = (w.abs() * ddct[:, None])[there]
    big_y = y.abs() * (i1 * (v1.abs() + (cn * m1).abs()))[:, None]
    adds = (t / 148 + 400) * 2.0 ** -24  # of a column sum: tokens of a block, then blocks

    def column(a, da, b, db):
        return (a * b).sum(0), (da * b.abs() + a.abs() * db + adds * (a * b).abs()).sum(0)

    checks = dict(
        d_residual=(i.scale * dr, abs(i.scale) * ddr, half),
        d_yp=(want_y, err_y, half),
        d_w=((dct[:, None] * y).sum(2), (ddct[:, None] * y.abs() + u * big_y).sum(2), 0.0),
        d_post=(*column(dr * gate, ddr * gate.abs(), cn, dcn), 0.0),
        d_gate=(*column(dr, ddr, cn * post, dcn * post.abs()), 0.0),
        d_pre=(*column(dn, u * dn.abs(), rn, drn), 0.0))
    for name, (want, err, step) in checks.items():
        g = got[name].double()
        if name == "d_yp":
            assert bool((g[~named] == 7.0).all())
            g, want, err = g[named], want[named], err[named]
        assert bool(((g - want).abs() <= 2 * err + step * want.abs() + 2.0 ** -100).all()), name


# Rows of one element to a few, many of them in a granule, and some of each width.
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(700001, 2, 1), (90001, 2, 7), (2500, 2, 1), (2501, 3, 2),
                                   (1301, 16, 17), (601, 2, 4096), (599, 3, 4095), (300, 1, 8192),
                                   (5, 2, 200)], ids=str)
def test_gradient_elementwise(cuda, shape, dtype):
    i = Inputs(*shape, dtype, cuda, 91, skip=True)
    out, normed, inv = i.forward()
    check_forward(i, out, normed, dtype)
    check_gradient_elementwise(i, i.backward(inv), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(9, 2, 200), (1701, 2, 4096), (601, 2, 512), (1650, 2, 1027),
                                   (700, 5, 520)], ids=str)
def test_tokens_without_routes(cuda, shape, dtype):
    """A padded batch: whole tokens, the first and last among them, whose routes went
    nowhere. c is zero there, r' the scaled residual, and no weight has a gradient."""
    i = Inputs(*shape, dtype, cuda, 92)
    idle = torch.arange(0, shape[0], 4, device=cuda)
    i.pos[idle], i.pos[-1] = -1, shape[0] * shape[1]
    out, normed, inv = i.forward()
    check_forward(i, out, normed, dtype)
    got = i.backward(inv)
    check_backward(i, got, dtype)
    assert torch.equal(out[idle], (i.scale * i.res[idle].float()).to(dtype))
    assert not got["d_w"][idle].any() and not got["d_w"][-1].any()
