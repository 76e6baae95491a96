"""rr_grouped_gated_gemm and its backward pass against float64.

Error bounds. A product of K terms accumulated in FP32 is within
4 K 2^-24 sum|x||w| of the exact one (the bound of the grouped GEMM); the
activation and the product add a few FP32 roundings; the output is rounded once
(half a step of its type). Normwise, one rounding to bfloat16 is at most
2^-8 / sqrt(3) of the result (uniform in a step, at the worst place of a
binade), two independent ones (the gradients' operands and results) sqrt(2) of
that; FP32 results are held to 2^-19: four truncated accumulations per 64-deep
block and one FP32 addition per block stay below 2^-20 for one product, and h
and the gradients combine two.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import raggedroute_b200 as rr
from expert_block_reference import (ACTIVATIONS, act, gated, gated_backward, half_step, magnitudes,
                                    normwise, offsets_of, random)

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32

# (segment lengths, rows behind the last segment, K, N): single rows and empty
# experts, lengths around the 64-, 128- and 256-row tiles, sizes that are no
# multiple of 8, and sizes of several tiles in every direction.
SHAPES = [
    ([1], 0, 1, 1),
    ([0, 1, 0], 0, 8, 8),
    ([2, 0, 3, 1], 1, 33, 17),
    ([5, 4, 0, 9], 0, 64, 32),
    ([33, 31, 1], 2, 72, 40),
    ([64, 65, 63, 0, 1], 3, 130, 129),
    ([127, 128, 129], 0, 128, 128),
    ([0, 257, 0, 255], 7, 200, 264),
    ([300, 1, 513], 5, 320, 384),
    ([700], 0, 1001, 333),
    ([40] * 37, 0, 96, 48),
]


# Long contractions and many tiles: two row blocks share a tile. Segments that
# end in each quarter of such a tile; N and K that end inside one.
LARGE = [
    ([700, 0, 1100, 257, 513, 130, 385, 1], 3, 2050, 3400),  # forward (contraction K)
    ([513, 900, 0, 1281, 100], 0, 3330, 1030),               # input gradient (2 N)
    ([2600, 4100], 5, 1100, 7700),                           # weight gradients (rows)
]
SHAPES += LARGE


def make(counts, behind, k, n, dtype, device, seed=0):
    rows = int(np.sum(counts)) + behind
    e = len(counts)
    x = random((rows, k), seed + 1, device, dtype)
    wg = random((e, k, n), seed + 2, device, dtype, 1 / math.sqrt(k))
    wu = random((e, k, n), seed + 3, device, dtype, 1 / math.sqrt(k))
    dh = random((rows, n), seed + 4, device, dtype)
    return x, wg, wu, offsets_of(counts, device), dh


def workspace(x, wg, backward=True):
    size = rr.grouped_gated_gemm_workspace_size(x.shape[0], *wg.shape, x.dtype, backward=backward)
    return torch.full((max(size, 256),), 0xCD, dtype=torch.uint8, device=x.device)


def forward(x, wg, wu, off, activation="silu", save=True, ws=None, ctx=None):
    rows, n = x.shape[0], wg.shape[2]
    h = torch.full((rows, n), 777.0, dtype=x.dtype, device=x.device)
    gu = torch.full((rows, 2 * n), 777.0, dtype=FP32, device=x.device) if save else None
    rr.grouped_gated_gemm(x, wg, wu, off, h, gate_up=gu, activation=activation,
                          workspace=workspace(x, wg) if ws is None else ws, ctx=ctx)
    return h, gu


def backward(x, wg, wu, off, gu, dh, activation="silu", ws=None, ctx=None):
    dx = torch.full_like(x, 777.0)
    dwg, dwu = torch.full_like(wg, 777.0), torch.full_like(wu, 777.0)
    rr.grouped_gated_gemm_backward(x, wg, wu, off, gu, dh, dx, dwg, dwu, activation=activation,
                                   workspace=workspace(x, wg) if ws is None else ws, ctx=ctx)
    return dx, dwg, dwu


def no_device_error():
    import ctypes
    from raggedroute_b200._lib import lib
    word = ctypes.c_uint32()
    lib().rr_consume_device_error(None, ctypes.byref(word))
    assert word.value == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(cuda, shape, dtype):
    counts, behind, k, n = shape
    x, wg, wu, off, _ = make(counts, behind, k, n, dtype, cuda)
    rows = int(np.sum(counts))
    if behind:
        x[rows:] = float("nan")
    h, gu = forward(x, wg, wu, off)
    no_device_error()
    g, u, want = gated(x, wg, wu, off)
    unit = 4 * k * 2.0 ** -24
    eg, eu = unit * magnitudes(x, wg, off), unit * magnitudes(x, wu, off)
    got_g, got_u = gu[:rows, :n].double(), gu[:rows, n:].double()
    assert bool(((got_g - g[:rows]).abs() <= eg[:rows] + 2.0 ** -24 * g[:rows].abs()).all())
    assert bool(((got_u - u[:rows]).abs() <= eu[:rows] + 2.0 ** -24 * u[:rows].abs()).all())
    # |silu'| <= 1.1; expf, the division and two products: under 16 FP32 steps.
    tol = (half_step(dtype) + 2.0 ** -20) * want.abs() + \
        1.1 * eg * (u.abs() + eu) + (act("silu", g).abs() + 2.0 ** -149) * eu
    assert bool(((h.double() - want).abs()[:rows] <= tol[:rows]).all())
    if k * n > 64:
        assert normwise(h[:rows], want[:rows]) < (2.0 ** -8 / math.sqrt(3) if dtype == BF16
                                                  else 2.0 ** -19)
    assert bool((h[rows:] == 777.0).all()) and bool((gu[rows:] == 777.0).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(cuda, shape, dtype):
    counts, behind, k, n = shape
    x, wg, wu, off, dh = make(counts, behind, k, n, dtype, cuda, seed=50)
    rows = int(np.sum(counts))
    if behind:
        x[rows:], dh[rows:] = float("nan"), float("inf")
    _, gu = forward(x, wg, wu, off)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh)
    no_device_error()
    assert bool((dx[rows:] == 777.0).all())
    want = gated_backward(x[:rows], wg, wu, off, dh[:rows])
    bound = math.sqrt(2) * 2.0 ** -8 / math.sqrt(3) if dtype == BF16 else 2.0 ** -19
    # Elementwise, against the sums of the products' magnitudes: dg, du and the
    # result carry a rounding each. dg = dh u silu'(g) and du = dh silu(g) also
    # carry the errors eg, eu of g and u, which are relative to sum|x||w| and not
    # to g or u where those cancel: with |silu'| <= 1.1 and |silu''| <= 0.5,
    #   |error of dg| <= |dh| (1.1 eu + 0.5 |u| eg), |error of du| <= 1.1 |dh| eg,
    # which enter the products beside dg and du (divided by rel, to share its
    # factor below).
    rel = 2 * half_step(dtype) + 2.0 ** -18 + 8 * max(k, n, rows) * 2.0 ** -24
    unit = 4 * k * 2.0 ** -24
    eg, eu = (unit * magnitudes(x[:rows], w, off) for w in (wg, wu))
    u = gated(x[:rows], wg, wu, off)[1].abs()
    d = dh[:rows].double().abs()
    dg = want[3].abs() + d * (1.1 * eu + 0.5 * u * eg) / rel
    du = want[4].abs() + 1.1 * d * eg / rel
    scale_x = torch.zeros_like(want[0])
    o = off.tolist()
    for e, (i, j) in enumerate(zip(o, o[1:])):
        scale_x[i:j] = dg[i:j] @ wg[e].double().abs().T + du[i:j] @ wu[e].double().abs().T
        sw = x[i:j].double().abs().T @ dg[i:j], x[i:j].double().abs().T @ du[i:j]
        for got, ref, s in ((dwg[e], want[1][e], sw[0]), (dwu[e], want[2][e], sw[1])):
            assert bool(((got.double() - ref).abs() <= rel * s + 2.0 ** -40).all())
    assert bool(((dx[:rows].double() - want[0]).abs() <= rel * scale_x + 2.0 ** -40).all())
    if k * n > 64:
        assert normwise(dx[:rows], want[0]) < bound
        assert normwise(dwg, want[1]) < bound and normwise(dwu, want[2]) < bound
    for e, c in enumerate(counts):
        if c == 0:
            assert not dwg[e].any() and not dwu[e].any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("rows", [3, 400])
def test_activations(cuda, activation, dtype, rows):
    x, wg, wu, off, dh = make([rows], 0, 64, 48, dtype, cuda, seed=9)
    wg = wg * 3
    h, gu = forward(x, wg, wu, off, activation)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh, activation)
    want = gated(x, wg, wu, off, activation)[2]
    ref = gated_backward(x, wg, wu, off, dh, activation)
    one = 2.0 ** -8 / math.sqrt(3) if dtype == BF16 else 2.0 ** -19
    two = math.sqrt(2) * one if dtype == BF16 else one
    assert normwise(h, want) < one
    assert normwise(dx, ref[0]) < two
    assert normwise(dwg, ref[1]) < two and normwise(dwu, ref[2]) < two


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_gradient_against_differences(cuda, activation):
    """<gradient, direction> equals the central difference of <h, dh> in float64."""
    x, wg, wu, off, dh = make([30, 0, 70], 0, 40, 24, FP32, cuda, seed=3)
    _, gu = forward(x, wg, wu, off, activation)
    grads = backward(x, wg, wu, off, gu, dh, activation)
    args = [x.double(), wg.double(), wu.double()]
    eps = 1e-5
    for i, grad in enumerate(grads):
        v = random(args[i].shape, 70 + i, cuda).double()
        values = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * eps * v
            values.append((gated(*moved, off, activation)[2] * dh.double()).sum())
        difference = float(values[0] - values[1]) / (2 * eps)
        # FP32 gradient: 2^-19 normwise; the difference itself: eps^2 terms.
        slack = float(2.0 ** -19 * grad.double().norm() * v.norm()) + 1e-6 * abs(difference)
        assert abs(float((grad.double() * v).sum()) - difference) <= slack


def test_parts_that_are_not_wanted(cuda):
    x, wg, wu, off, dh = make([40, 60], 0, 64, 64, BF16, cuda, seed=5)
    _, gu = forward(x, wg, wu, off)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh)
    ws = workspace(x, wg)
    dx2 = torch.zeros_like(dx)
    rr.grouped_gated_gemm_backward(x, wg, wu, off, gu, dh, dx2, None, None, workspace=ws)
    dwg2, dwu2 = torch.zeros_like(dwg), torch.zeros_like(dwu)
    rr.grouped_gated_gemm_backward(x, wg, wu, off, gu, dh, None, dwg2, dwu2, workspace=ws)
    assert torch.equal(dx, dx2) and torch.equal(dwg, dwg2) and torch.equal(dwu, dwu2)
    h, _ = forward(x, wg, wu, off)
    h2, _ = forward(x, wg, wu, off, save=False)
    assert torch.equal(h, h2)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_other_segments_do_not_leak(cuda, dtype):
    """Infinities and NaN in one expert's rows stay out of the others'."""
    counts = [70, 90, 65]
    x, wg, wu, off, dh = make(counts, 0, 72, 56, dtype, cuda, seed=11)
    _, gu = forward(x, wg, wu, off)
    clean = backward(x, wg, wu, off, gu, dh)
    x2, dh2 = x.clone(), dh.clone()
    x2[70:160:2] = float("inf")
    x2[71:160:2] = float("nan")
    dh2[70:160] = float("nan")
    h2, gu2 = forward(x2, wg, wu, off)
    dirty = backward(x2, wg, wu, off, gu2, dh2)
    for rows in (slice(0, 70), slice(160, 225)):
        assert torch.equal(dirty[0][rows], clean[0][rows])
    for e in (0, 2):
        assert torch.equal(dirty[1][e], clean[1][e]) and torch.equal(dirty[2][e], clean[2][e])
    assert not torch.isfinite(h2[70:160]).any()
    assert not torch.isfinite(dirty[1][1]).any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [4, 700])
def test_saturated_activation(cuda, dtype, rows):
    """Gates far out in both directions: exp overflows and underflows."""
    x = torch.ones(rows, 8, dtype=dtype, device=cuda)
    wg = torch.zeros(1, 8, 16, dtype=dtype, device=cuda)
    wg[0, 0] = torch.linspace(-400, 400, 16).to(cuda, dtype)
    wu = torch.full_like(wg, 0.125)
    off = offsets_of([rows], cuda)
    h, gu = forward(x, wg, wu, off)
    want = gated(x, wg, wu, off)[2]
    assert torch.isfinite(h).all()
    assert bool(((h.double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-30).all())
    dx, dwg, dwu = backward(x, wg, wu, off, gu, torch.ones_like(h))
    assert all(torch.isfinite(t).all() for t in (dx, dwg, dwu))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_repeats_bit_for_bit_and_replays(cuda, dtype):
    """Equal results in a second call, on another stream, and in a captured
    graph replayed on new inputs; two graphs may share the workspace."""
    shape = ([90, 0, 200, 33], 0, 136, 72)
    x, wg, wu, off, dh = make(*shape, dtype, cuda, seed=20)
    ws = workspace(x, wg)
    first = forward(x, wg, wu, off, ws=ws)
    grads = backward(x, wg, wu, off, first[1], dh, ws=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = forward(x, wg, wu, off, ws=ws)
        grads2 = backward(x, wg, wu, off, again[1], dh, ws=ws)
    side.synchronize()
    for a, b in zip(first + grads, again + grads2):
        assert torch.equal(a, b)
    h, gu = torch.zeros_like(first[0]), torch.zeros_like(first[1])
    out = [torch.zeros_like(t) for t in grads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    bufs = [t.clone() for t in (x, off, dh)]

    def train(ctx):
        rr.grouped_gated_gemm(bufs[0], wg, wu, bufs[1], h, gate_up=gu, workspace=ws, ctx=ctx)
        rr.grouped_gated_gemm_backward(bufs[0], wg, wu, bufs[1], gu, bufs[2], *out, workspace=ws,
                                       ctx=ctx)

    def serve(ctx):
        rr.grouped_gated_gemm(bufs[0], wg, wu, bufs[1], h, workspace=ws, ctx=ctx)

    torch.cuda.synchronize()
    graphs = [rr.Graph.capture(train, s), rr.Graph.capture(serve, s)]
    x2, _, _, off2, dh2 = make([0, 300, 23, 0], 0, 136, 72, dtype, cuda, seed=33)
    for xs, offs, ds in ((x, off, dh), (x2, off2, dh2)):
        want = forward(xs, wg, wu, offs)
        want_grads = backward(xs, wg, wu, offs, want[1], ds)
        for dst, src in zip(bufs, (xs, offs, ds)):
            dst.copy_(src)
        torch.cuda.synchronize()
        graphs[0].launch(s)
        s.synchronize()
        assert torch.equal(h, want[0]) and all(torch.equal(a, b) for a, b in zip(out, want_grads))
        h.zero_()
        torch.cuda.synchronize()
        graphs[1].launch(s)
        s.synchronize()
        assert torch.equal(h, want[0])
    no_device_error()


def test_clipped_offsets(cuda):
    """Offsets that reach past the rows, or fall, touch nothing outside them."""
    x, wg, wu, _, dh = make([500], 0, 64, 64, BF16, cuda, seed=40)
    wg, wu = wg.expand(3, 64, 64).contiguous(), wu.expand(3, 64, 64).contiguous()
    guard = torch.full((700, 64), 5.0, dtype=BF16, device=cuda)
    off = torch.tensor([-7, 200, 150, 100000], dtype=torch.int32, device=cuda)
    rr.grouped_gated_gemm(x, wg, wu, off, guard[:500], workspace=workspace(x, wg))
    torch.cuda.synchronize()
    assert bool((guard[500:] == 5.0).all())
    want = gated(x, wg[:1], wu[:1], offsets_of([500], cuda))[2]
    assert normwise(guard[:500], want) < 2.0 ** -8 / math.sqrt(3)
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_buffers_at_odd_addresses(cuda, dtype):
    """Odd rows may start anywhere; canaries around every output stay."""
    x, wg, wu, off, dh = make([50, 21], 0, 35, 21, dtype, cuda, seed=60)

    def odd(t):
        flat = torch.full((t.numel() + 130,), 9.0, dtype=t.dtype, device=cuda)
        view = flat[65:65 + t.numel()].view(t.shape)
        return flat, view.copy_(t)

    xs, gs, us, ds = (odd(t)[1] for t in (x, wg, wu, dh))
    want_h, want_gu = forward(x, wg, wu, off)
    want = backward(x, wg, wu, off, want_gu, dh)
    hf, h = odd(torch.zeros_like(want_h))
    gf, gu = odd(torch.zeros_like(want_gu))
    outs = [odd(torch.zeros_like(t)) for t in want]
    ws = workspace(x, wg)
    rr.grouped_gated_gemm(xs, gs, us, off, h, gate_up=gu, workspace=ws)
    rr.grouped_gated_gemm_backward(xs, gs, us, off, gu, ds, *(v for _, v in outs), workspace=ws)
    assert torch.equal(h, want_h) and torch.equal(gu, want_gu)
    for (flat, view), t in zip(outs + [(hf, h)], list(want) + [want_h]):
        assert torch.equal(view, t)
        assert bool((flat[:65] == 9.0).all()) and bool((flat[65 + t.numel():] == 9.0).all())


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 31, 32, 33, 34])
def test_one_form_meets_the_other(cuda, rows):
    """The few-row and the tensor-core forms agree around their boundary."""
    x, wg, wu, off, _ = make([rows], 0, 512, 256, BF16, cuda, seed=80)
    h, _ = forward(x, wg, wu, off)
    assert normwise(h, gated(x, wg, wu, off)[2]) < 2.0 ** -8 / math.sqrt(3)


@pytest.mark.parametrize("dtype,k,n,experts,rows", [
    (BF16, 64, 48, 40, 10), (BF16, 64, 48, 40, 11), (BF16, 63, 48, 6, 24), (BF16, 63, 48, 6, 25),
    (FP32, 64, 48, 6, 48), (FP32, 64, 48, 6, 49)])
def test_backward_forms_meet(cuda, dtype, k, n, experts, rows):
    """Both sides of each boundary between the backward pass's two forms."""
    counts = np.random.default_rng(rows).multinomial(rows, [1 / experts] * experts)
    x, wg, wu, off, dh = make(counts, 2, k, n, dtype, cuda, seed=81)
    _, gu = forward(x, wg, wu, off)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh)
    want = gated_backward(x[:rows], wg, wu, off, dh[:rows])
    bound = math.sqrt(2) * 2.0 ** -8 / math.sqrt(3) if dtype == BF16 else 2.0 ** -19
    for got, ref in zip((dx[:rows], dwg, dwu), want):
        assert normwise(got, ref) < bound
    assert bool((dx[rows:] == 777.0).all())


def test_many_experts(cuda):
    counts = np.random.default_rng(1).integers(0, 4, 1024)
    x, wg, wu, off, dh = make(counts, 0, 16, 16, FP32, cuda, seed=90)
    h, gu = forward(x, wg, wu, off)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh)
    want = gated_backward(x, wg, wu, off, dh)
    assert normwise(h, gated(x, wg, wu, off)[2]) < 2.0 ** -19
    assert normwise(dx, want[0]) < 2.0 ** -19 and normwise(dwg, want[1]) < 2.0 ** -19
    assert normwise(dwu, want[2]) < 2.0 ** -19


def test_no_rows(cuda):
    x, wg, wu, off, dh = make([0, 0], 0, 16, 8, BF16, cuda)
    h, gu = forward(x, wg, wu, off)
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh)
    assert h.numel() == 0 and dx.numel() == 0 and not dwg.any() and not dwu.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shift", range(1, 8))
def test_buffers_that_start_anywhere(cuda, dtype, shift):
    """Rows of no multiple of 16 bytes from buffers that start at any element,
    between values that are not theirs: the same bits as from aligned copies."""
    e, r, k, n = 3, 300, 131, 53

    def moved(t):
        buf = torch.full((t.numel() + 16,), float("nan"), dtype=t.dtype, device=cuda)
        view = buf[shift:shift + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    x, dh = random((r, k), 1, cuda, dtype=dtype), random((r, n), 2, cuda, dtype=dtype)
    wg, wu = random((e, k, n), 3, cuda, dtype=dtype), random((e, k, n), 4, cuda, dtype=dtype)
    gu = random((r, 2 * n), 5, cuda)
    off = torch.tensor([0, 100, 100, r], dtype=torch.int32, device=cuda)
    size = rr.grouped_gated_gemm_workspace_size(r, e, k, n, dtype, backward=True)
    assert size > 0  # operands are packed
    results = []
    for place in (lambda t: t, moved):
        ws = torch.empty(size, dtype=torch.uint8, device=cuda)
        h, dx = torch.empty(r, n, dtype=dtype, device=cuda), torch.empty_like(x)
        dwg, dwu = torch.empty_like(wg), torch.empty_like(wu)
        rr.grouped_gated_gemm(place(x), place(wg), place(wu), off, h, workspace=ws)
        rr.grouped_gated_gemm_backward(place(x), place(wg), place(wu), off, place(gu), place(dh),
                                       dx, dwg, dwu, workspace=ws)
        results.append((h, dx, dwg, dwu))
    for a, b in zip(*results):
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()
