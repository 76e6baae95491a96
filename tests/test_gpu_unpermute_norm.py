"""rr_unpermute_norm and its backward pass against float64.

Error bounds. A row's sums are at most 16 terms per thread and ten levels of a
tree, of positive terms in the means: under 32 FP32 steps relative. With the
products around them every FP32 value stays within 64 * 2^-24 of the sum of its
terms' magnitudes (and top_k more for c); each output adds half a step of its
type.
"""
from __future__ import annotations

import math

import pytest
import torch

import raggedroute_b200 as rr
from expert_block_reference import half_step, normwise, random, unpermute_norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
EPS = 1e-6

# (tokens, top_k, output): one column to the widest row, either side of each
# block size, odd widths, and more tokens than the gradient has blocks.
SHAPES = [(1, 1, 1), (1, 2, 4096), (3, 2, 8), (5, 1, 33), (17, 8, 257), (64, 2, 512), (9, 3, 520),
          (33, 2, 1024), (7, 64, 96), (6, 2, 4100), (4, 2, 8191), (3, 2, 8192), (3, 1, 8200),
          (2, 2, 16384), (2, 2, 16383), (2500, 2, 64), (700, 4, 1000)]

# Enough tokens for the streamed form: each team size, rows that start on odd
# addresses in both types, many routes, and token counts that end inside a stage.
SHAPES += [(5001, 2, 96), (4800, 1, 511), (4738, 3, 333), (2400, 2, 1026), (1201, 16, 520),
           (700, 2, 2340), (601, 2, 4096), (599, 2, 4095), (299, 2, 8192), (300, 1, 8191),
           (297, 5, 6001)]


class Inputs:
    def __init__(self, tokens, top_k, output, dtype, device, seed=0, post=True, gate=True,
                 pre=True, skip=False):
        r = tokens * top_k
        g = torch.Generator(device=device).manual_seed(seed)
        self.pos = torch.randperm(r, generator=g, device=device).to(torch.int32).view(tokens, top_k)
        if skip:  # routes that went nowhere
            self.pos.view(-1)[::3] = torch.tensor([-1, r, 2 ** 31 - 1], dtype=torch.int32,
                                                  device=device).repeat(r)[:len(self.pos.view(-1)[::3])]
        self.w = torch.softmax(random((tokens, top_k), seed + 1, device), 1)
        self.yp = random((r, output), seed + 2, device, dtype, 0.5)
        self.res = random((tokens, output), seed + 3, device, dtype)
        self.post = random((output,), seed + 4, device, std=0.2) + 1 if post else None
        self.gate = random((output,), seed + 5, device, std=0.5) if gate else None
        self.pre = random((output,), seed + 6, device, std=0.2) + 1 if pre else None
        self.dro = random((tokens, output), seed + 7, device, dtype)
        self.dn = random((tokens, output), seed + 8, device, dtype) if pre else None
        self.scale = 0.75

    def leaves(self):
        return [None if t is None else t.double().requires_grad_()
                for t in (self.yp, self.w, self.res, self.post, self.gate, self.pre)]

    def forward(self, ctx=None, out=None):
        out = torch.empty_like(self.res) if out is None else out
        normed = None if self.pre is None else torch.empty_like(self.res)
        inv = torch.empty(self.res.shape[0], 2, device=self.res.device)
        rr.unpermute_norm(self.yp, self.pos, self.w, self.res, out, normed, post_gamma=self.post,
                          gate=self.gate, pre_gamma=self.pre, inv_rms=inv, eps=EPS,
                          residual_scale=self.scale, ctx=ctx)
        return out, normed, inv

    def backward(self, inv, ctx=None, ws=None, d_residual=None):
        t, n = self.res.shape
        dev = self.res.device
        g = dict(d_residual=torch.full_like(self.res, 7.0) if d_residual is None else d_residual,
                 d_yp=torch.full_like(self.yp, 7.0), d_w=torch.full_like(self.w, 7.0))
        for name, p in (("d_post", self.post), ("d_gate", self.gate), ("d_pre", self.pre)):
            g[name] = None if p is None else torch.full((n,), 7.0, device=dev)
        if ws is None:
            size = rr.unpermute_norm_backward_workspace_size(t, n)
            ws = torch.full((max(size, 256),), 0xCD, dtype=torch.uint8, device=dev)
        rr.unpermute_norm_backward(self.yp, self.pos, self.w, self.res, inv, self.dro, self.dn,
                                   g["d_residual"], g["d_yp"], g["d_w"], post_gamma=self.post,
                                   gate=self.gate, pre_gamma=self.pre, d_post_gamma=g["d_post"],
                                   d_gate=g["d_gate"], d_pre_gamma=g["d_pre"],
                                   residual_scale=self.scale, workspace=ws, ctx=ctx)
        return g


def check_forward(i: Inputs, out, normed, dtype):
    yp, w, res, post, gate, pre = i.leaves()
    want, want_n = unpermute_norm(yp, i.pos, w, res, post, gate, pre, EPS, i.scale)
    # The magnitudes: b from sum |w||v|, r' from scale |residual| + |gate b|.
    big, _ = unpermute_norm(yp.abs(), i.pos, w.abs(), res.abs() * 0, None, None, None, EPS, 0.0)
    if post is not None:
        c, _ = unpermute_norm(yp, i.pos, w, res * 0, None, None, None, EPS, 0.0)
        big = big / torch.sqrt((c * c).mean(1, keepdim=True) + EPS) * post.abs()
    if gate is not None:
        big = big * gate.abs()
    unit = (64 + i.pos.shape[1]) * 2.0 ** -24
    err = unit * (abs(i.scale) * res.abs() + 2 * big)
    assert bool(((out.double() - want).abs() <= half_step(dtype) * want.abs() + err).all())
    if pre is not None:
        i2 = 1 / torch.sqrt((want * want).mean(1, keepdim=True) + EPS)
        # i2 moves with the errors of the whole row: at most their rms over r's.
        drift = (err * err).mean(1, keepdim=True).sqrt() * i2
        tol = (half_step(dtype) + unit + drift) * want_n.abs() + err * i2 * pre.abs()
        assert bool(((normed.double() - want_n).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(cuda, shape, dtype):
    i = Inputs(*shape, dtype, cuda)
    out, normed, _ = i.forward()
    check_forward(i, out, normed, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("parts", [(0, 0, 0), (0, 1, 1), (1, 0, 1), (1, 1, 0), (0, 0, 1)])
def test_parts(cuda, parts, dtype):
    post, gate, pre = map(bool, parts)
    for shape in ((21, 2, 200), (4, 3, 77)):
        i = Inputs(*shape, dtype, cuda, 40, post=post, gate=gate, pre=pre, skip=True)
        out, normed, inv = i.forward()
        check_forward(i, out, normed, dtype)
        check_backward(i, i.backward(inv), dtype)


def check_backward(i: Inputs, got, dtype):
    leaves = i.leaves()
    yp, w, res, post, gate, pre = leaves
    want_r, want_n = unpermute_norm(yp, i.pos, w, res, post, gate, pre, EPS, i.scale)
    outs, grads = [want_r], [i.dro.double()]
    if want_n is not None:
        outs.append(want_n)
        grads.append(i.dn.double())
    given = [t for t in leaves if t is not None]
    named = dict(zip([n for n, t in zip(("d_yp", "d_w", "d_residual", "d_post", "d_gate", "d_pre"),
                                        leaves) if t is not None],
                     torch.autograd.grad(outs, given, grads)))
    routes = i.yp.shape[0]
    named_rows = torch.zeros(routes, dtype=torch.bool, device=i.yp.device)
    p = i.pos.view(-1).long()
    p = p[(p >= 0) & (p < routes)]
    named_rows[p] = True
    # Rows that no route names are left as they were.
    assert bool((got["d_yp"][~named_rows] == 7.0).all())
    one = half_step(dtype) / math.sqrt(3) + 2.0 ** -19
    # With one route per token and a norm of c, d_w is exactly the part of the
    # gradient that the norm removes: zero up to eps, lost in rounding.
    tiny = i.pos.shape[1] == 1 and post is not None
    narrow = i.res.shape[1] < 8  # the norm leaves next to nothing of a row's gradient
    for name, want in named.items():
        g = got[name].double()
        if name == "d_yp":
            g, want = g[named_rows], want[named_rows]
        if name == "d_w" and tiny or narrow:
            scale = max(1.0, float(i.dro.double().abs().max())) * 64
            assert bool(((g - want).abs() <= 2.0 ** -8 * scale).all()), name
            continue
        assert normwise(g, want) < (one if got[name].dtype == dtype and dtype == BF16
                                    else 2.0 ** -19), name


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(cuda, shape, dtype):
    i = Inputs(*shape, dtype, cuda, seed=90)
    _, _, inv = i.forward()
    first = i.backward(inv)
    check_backward(i, first, dtype)
    second = i.backward(inv)
    for name, t in first.items():
        assert torch.equal(t, second[name]), name


def test_gradient_against_differences(cuda):
    """<gradient, direction> equals the float64 central difference."""
    i = Inputs(12, 2, 96, FP32, cuda, seed=17)
    _, _, inv = i.forward()
    got = i.backward(inv)
    leaves = [t.detach() for t in i.leaves()]
    eps = 1e-6
    for k, name in enumerate(("d_yp", "d_w", "d_residual", "d_post", "d_gate", "d_pre")):
        v = random(leaves[k].shape, 200 + k, cuda).double()
        values = []
        for sign in (1, -1):
            a = list(leaves)
            a[k] = leaves[k] + sign * eps * v
            r, n = unpermute_norm(a[0], i.pos, a[1], a[2], a[3], a[4], a[5], EPS, i.scale)
            values.append(float((r * i.dro.double()).sum() + (n * i.dn.double()).sum()))
        difference = (values[0] - values[1]) / (2 * eps)
        slack = float(2.0 ** -19 * got[name].double().norm() * v.norm()) + 1e-6 * abs(difference)
        assert abs(float((got[name].double() * v).sum()) - difference) <= slack, name


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_in_place_and_missing_gradients(cuda, dtype):
    i = Inputs(40, 2, 264, dtype, cuda, seed=3)
    out, normed, inv = i.forward()
    want = i.backward(inv)
    d = i.dro.clone()
    keep = i.dro
    i.dro = d
    got = i.backward(inv, d_residual=d)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    i.dro = keep
    res = i.res.clone()
    i.res = res
    out2, normed2, _ = i.forward(out=res)
    assert torch.equal(out, out2) and torch.equal(normed, normed2)
    # No gradient into normed: the block's norm takes no part.
    j = Inputs(40, 2, 264, dtype, cuda, seed=3)
    _, _, inv = j.forward()
    dn, j.dn = j.dn, None
    a = j.backward(inv)
    assert not a["d_pre"].any()
    j.dn = torch.zeros_like(dn)
    b = j.backward(inv)
    assert normwise(a["d_residual"], b["d_residual"]) < 2.0 ** -20 + half_step(dtype)
    # No gradient into residual_out: as if it were zero.
    j.dn, j.dro = dn, None
    c = j.backward(inv)
    j.dro = torch.zeros_like(dn)
    e = j.backward(inv)
    for name in c:
        assert torch.equal(c[name], e[name]), name


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_buffers_at_odd_addresses(cuda, dtype):
    """The vector and the scalar form agree; canaries stay."""
    i = Inputs(10, 2, 512, dtype, cuda, seed=6)
    out, normed, inv = i.forward()
    flat = torch.full((out.numel() + 258,), 9.0, dtype=dtype, device=cuda)
    view = flat[129:129 + out.numel()].view(out.shape)
    out2, normed2, inv2 = i.forward(out=view)
    assert normwise(out2, out.double()) < 2 * half_step(dtype)
    assert normwise(inv2, inv.double()) < 2.0 ** -20
    assert bool((flat[:129] == 9.0).all()) and bool((flat[129 + out.numel():] == 9.0).all())
    check_forward(i, out2, normed2, dtype)


def test_not_finite_tokens_stay_alone(cuda):
    i = Inputs(6, 2, 128, FP32, cuda, seed=8)
    out, normed, _ = i.forward()
    i.yp[int(i.pos[2, 0])] = float("nan")
    i.res[4, 7] = float("inf")
    out2, normed2, _ = i.forward()
    for t in (0, 1, 3, 5):
        assert torch.equal(out[t], out2[t]) and torch.equal(normed[t], normed2[t])
    assert torch.isnan(out2[2]).all() and torch.isinf(out2[4, 7])


def test_replay_and_stream(cuda):
    i = Inputs(300, 2, 640, BF16, cuda, seed=12)
    out, normed = torch.empty_like(i.res), torch.empty_like(i.res)
    inv = torch.empty(300, 2, device=cuda)
    ws = torch.empty(rr.unpermute_norm_backward_workspace_size(300, 640), dtype=torch.uint8,
                     device=cuda)
    g = dict(d_residual=torch.empty_like(i.res), d_y_permuted=torch.empty_like(i.yp),
             d_route_weights=torch.empty_like(i.w))
    p = dict(d_post_gamma=torch.empty(640, device=cuda), d_gate=torch.empty(640, device=cuda),
             d_pre_gamma=torch.empty(640, device=cuda))

    def step(ctx):
        rr.unpermute_norm(i.yp, i.pos, i.w, i.res, out, normed, post_gamma=i.post, gate=i.gate,
                          pre_gamma=i.pre, inv_rms=inv, eps=EPS, ctx=ctx)
        rr.unpermute_norm_backward(i.yp, i.pos, i.w, i.res, inv, i.dro, i.dn, *g.values(),
                                   post_gamma=i.post, gate=i.gate, pre_gamma=i.pre, **p,
                                   workspace=ws, ctx=ctx)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = rr.Graph.capture(step, s)
    for seed in (1, 2):
        i.yp.copy_(random(i.yp.shape, seed, cuda, BF16))
        torch.cuda.synchronize()
        graph.launch(s)
        s.synchronize()
        got = [t.clone() for t in (out, normed, inv, *g.values(), *p.values())]
        step(None)
        torch.cuda.synchronize()
        for a, b in zip(got, (out, normed, inv, *g.values(), *p.values())):
            assert torch.equal(a, b)


# Enough bytes for the streamed forward pass: each team size, both alignments, many
# routes, token counts that end inside a stage.
STREAMED = [(13201, 2, 512), (6600, 2, 1000), (3299, 2, 2048), (1701, 2, 4096), (901, 2, 8192),
            (1001, 16, 2056), (21000, 1, 130), (8003, 3, 333), (1650, 2, 1027), (421, 2, 8191)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", STREAMED, ids=str)
def test_streamed_forward(cuda, shape, dtype):
    i = Inputs(*shape, dtype, cuda, seed=31, skip=shape[1] > 1)
    out, normed, inv = i.forward()
    check_forward(i, out, normed, dtype)
    again = i.forward()
    assert all(torch.equal(a, b) for a, b in zip((out, normed, inv), again))
    i.res = i.res.clone()
    out2, normed2, inv2 = i.forward(out=i.res)  # in place
    assert torch.equal(out, out2) and torch.equal(normed, normed2) and torch.equal(inv, inv2)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(1, 2, 515), (2, 4, 178), (149, 2, 512), (148, 1, 4096),
                                   (1185, 2, 120), (297, 2, 8192)], ids=str)
def test_streamed_gradient_of_few_tokens(cuda, shape, dtype):
    """Fewer tokens than teams: most of a block has none."""
    i = Inputs(*shape, dtype, cuda, seed=47)
    _, _, inv = i.forward()
    first = i.backward(inv)
    check_backward(i, first, dtype)
    second = i.backward(inv)
    assert all(torch.equal(t, second[name]) for name, t in first.items())
