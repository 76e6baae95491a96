"""rr_grouped_gated_gemm and its backward pass in FP32 where the tensor-core form
runs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_b200 as rr
from expert_block_reference import ACTIVATIONS, gated, gated_backward, normwise, offsets_of
from test_gpu_gated import FP32, backward, forward, make, no_device_error, workspace

pytestmark = pytest.mark.gpu

LONG = 0x3F80FFFF  # 1 + 65535 * 2^-23: rounds down to 8 bits with the longest remainder


def takes_tensor_cores(x, wg, wu, off) -> bool:
    """Whether the forward call needs its operands packed, which only that form does."""
    h = torch.empty(x.shape[0], wg.shape[2], dtype=x.dtype, device=x.device)
    try:
        rr.grouped_gated_gemm(x, wg, wu, off, h)
    except rr.RaggedRouteError as e:
        assert e.code == rr.StatusCode.INSUFFICIENT_WORKSPACE
        return True
    return False


def long_mantissas(shape, seed, device):
    """Values in [1, 2) of 24 significant bits, the worst one first."""
    g = torch.Generator(device=device).manual_seed(seed)
    bits = torch.randint(0, 1 << 23, shape, generator=g, device=device, dtype=torch.int32)
    bits |= 0x3F800001
    bits.view(-1)[0] = LONG
    return bits.view(torch.float32)


# One product. Its parts are exact, what the six part products leave out is
# at most 2^-24 of it, and the accumulator cuts the last sum twice, by alignment and
# by normalisation (2^-23 each); the sums before it are 2^-7 of it at most, five of
# them cut the same way.
ONE_PRODUCT = 2.0 ** -24 + 2 * 2.0 ** -23 * (1 + 5 * 2.0 ** -7)


def test_products_of_long_mantissas(cuda):
    """A single product per result, of operands of one sign."""
    x = long_mantissas((2000, 1), 1, cuda)
    wg, wu = long_mantissas((1, 1, 128), 2, cuda), -long_mantissas((1, 1, 128), 3, cuda)
    off = offsets_of([2000], cuda)
    assert takes_tensor_cores(x, wg, wu, off)
    _, gu = forward(x, wg, wu, off)
    no_device_error()
    want = x.double() @ torch.cat((wg, wu), 2)[0].double()
    assert float(((gu.double() - want) / want).abs().max()) <= ONE_PRODUCT


def test_gradients_of_long_mantissas(cuda):
    """The same for dx (one column) and dWg (one row with a gradient)."""
    rows, k = 64, 96
    x, wg = long_mantissas((rows, k), 4, cuda), long_mantissas((1, k, 1), 5, cuda)
    wu, off = torch.zeros_like(wg), offsets_of([rows], cuda)
    dh = torch.zeros(rows, 1, device=cuda)
    dh[0] = long_mantissas((1, 1), 6, cuda)
    gu = torch.ones(rows, 2, device=cuda)  # relu: dg = dh * up
    dx, dwg, dwu = backward(x, wg, wu, off, gu, dh, "relu")
    no_device_error()
    want = dh[0].double() * wg[0, :, 0].double()
    assert float(((dx[0].double() - want) / want).abs().max()) <= ONE_PRODUCT
    assert not dx[1:].any()
    want = dh[0].double() * x[0].double()
    for got in (dwg, dwu):
        assert float(((got[0, :, 0].double() - want) / want).abs().max()) <= ONE_PRODUCT


def test_products_of_any_magnitude(cuda):
    """Single products over the whole range of exponents, the largest floats (which do
    not round up to infinity) and subnormal ones among them. An operand below 2^-110
    is met within 2^-134; where the product is far above 2^-126, so are the parts'
    products that count."""
    g = torch.Generator(device=cuda).manual_seed(8)

    def operand(n):
        e = torch.randint(-140, 128, (n,), generator=g, device=cuda)
        m = 1 + torch.rand(n, generator=g, device=cuda, dtype=torch.float64)
        v = (m * 2.0 ** e.double()).clamp(max=torch.finfo(torch.float32).max).float()
        v[:4] = torch.tensor([torch.finfo(torch.float32).max, 2.0 ** -149, -1.0, 0.0])
        return v * (1 - 2 * torch.randint(0, 2, (n,), generator=g, device=cuda))

    x, wg, wu = operand(2000)[:, None], operand(128)[None, None], operand(128)[None, None]
    off = offsets_of([2000], cuda)
    assert takes_tensor_cores(x, wg, wu, off)
    _, gu = forward(x, wg, wu, off)
    no_device_error()
    w = torch.cat((wg, wu), 2)[0].double()
    want = x.double() @ w
    inside = (want.abs() > 2.0 ** -100) & (want.abs() < 2.0 ** 127)
    tol = ONE_PRODUCT * want.abs() + 2.0 ** -134 * (x.double().abs() + w.abs())
    assert int(inside.sum()) > 50000
    assert bool(((gu.double() - want).abs() <= tol)[inside].all())
    assert not torch.isfinite(gu[want.abs() > 2.0 ** 128]).any()
    assert bool((gu.double()[want.abs() < 2.0 ** -100].abs() <= 2.0 ** -99).all())


K, N = 520, 264  # the tensor-core form from a few hundred rows on


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_activations(cuda, activation):
    x, wg, wu, off, dh = make([700], 0, K, N, FP32, cuda, seed=9)
    wg = wg * 3
    assert takes_tensor_cores(x, wg, wu, off)
    h, gu = forward(x, wg, wu, off, activation)
    grads = backward(x, wg, wu, off, gu, dh, activation)
    assert normwise(h, gated(x, wg, wu, off, activation)[2]) < 2.0 ** -19
    for got, want in zip(grads, gated_backward(x, wg, wu, off, dh, activation)):
        assert normwise(got, want) < 2.0 ** -19


def test_other_segments_do_not_leak(cuda):
    """Infinities and NaN in one expert's rows and weights stay out of the others', and
    of the rows behind the last segment."""
    counts = [270, 290, 265]
    x, wg, wu, off, dh = make(counts, 9, K, N, FP32, cuda, seed=11)
    assert takes_tensor_cores(x, wg, wu, off)
    h, gu = forward(x, wg, wu, off)
    clean = backward(x, wg, wu, off, gu, dh)
    x2, dh2, wg2 = x.clone(), dh.clone(), wg.clone()
    x2[270:560:2], x2[271:560:2], x2[825:] = float("inf"), float("nan"), float("nan")
    dh2[270:560] = float("nan")
    wg2[1, 3] = float("inf")
    h2, gu2 = forward(x2, wg2, wu, off)
    dirty = backward(x2, wg2, wu, off, gu2, dh2)
    for rows in (slice(0, 270), slice(560, 825)):
        assert torch.equal(h2[rows], h[rows]) and torch.equal(gu2[rows], gu[rows])
        assert torch.equal(dirty[0][rows], clean[0][rows])
    for e in (0, 2):
        assert torch.equal(dirty[1][e], clean[1][e]) and torch.equal(dirty[2][e], clean[2][e])
    assert not torch.isfinite(h2[270:560]).any() and not torch.isfinite(dirty[1][1]).any()
    assert bool((h2[825:] == 777.0).all()) and bool((dirty[0][825:] == 777.0).all())


def test_saturated_activation(cuda):
    """Gates far out in both directions: exp overflows and underflows."""
    x = torch.ones(700, K, device=cuda)
    wg = torch.zeros(1, K, N, device=cuda)
    wg[0, 0] = torch.linspace(-400, 400, N).to(cuda)
    wu = torch.zeros_like(wg)
    wu[0, :8] = 0.125
    off = offsets_of([700], cuda)
    assert takes_tensor_cores(x, wg, wu, off)
    h, gu = forward(x, wg, wu, off)
    want = gated(x, wg, wu, off)[2]
    # The gate is exact in three parts; expf, the division and the product: 8 steps.
    assert bool(((h.double() - want).abs() <= 2.0 ** -21 * want.abs() + 1e-30).all())
    assert all(torch.isfinite(t).all() for t in backward(x, wg, wu, off, gu, torch.ones_like(h)))


def test_repeats_bit_for_bit_and_replays(cuda):
    """Equal results in a second call and in a captured graph replayed on new inputs."""
    x, wg, wu, off, dh = make([310, 0, 500, 33], 0, K, N, FP32, cuda, seed=20)
    assert takes_tensor_cores(x, wg, wu, off)
    ws = workspace(x, wg)
    h, gu = torch.zeros(843, N, device=cuda), torch.zeros(843, 2 * N, device=cuda)
    out = [torch.zeros_like(t) for t in (x, wg, wu)]
    bufs = [t.clone() for t in (x, off, dh)]

    def train(ctx):
        rr.grouped_gated_gemm(bufs[0], wg, wu, bufs[1], h, gate_up=gu, workspace=ws, ctx=ctx)
        rr.grouped_gated_gemm_backward(bufs[0], wg, wu, bufs[1], gu, bufs[2], *out, workspace=ws,
                                       ctx=ctx)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = rr.Graph.capture(train, s)
    x2, _, _, off2, dh2 = make([0, 800, 43, 0], 0, K, N, FP32, cuda, seed=33)
    for xs, offs, ds in ((x, off, dh), (x2, off2, dh2)):
        want = forward(xs, wg, wu, offs)
        want += backward(xs, wg, wu, offs, want[1], ds)
        again = forward(xs, wg, wu, offs)
        assert all(torch.equal(a, b) for a, b in zip(want, again))
        for dst, src in zip(bufs, (xs, offs, ds)):
            dst.copy_(src)
        torch.cuda.synchronize()
        for _ in range(2):
            graph.launch(s)
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((h, gu, *out), want))
    no_device_error()


@pytest.mark.parametrize("shift", range(1, 4))
def test_buffers_that_start_anywhere(cuda, shift):
    """Rows of no multiple of 16 bytes, packed from buffers that start at any element
    between values that are not theirs, into buffers between canaries."""
    k, n = K - 1, N - 1
    x, wg, wu, off, _ = make([400, 0, 500], 0, k, n, FP32, cuda, seed=60)
    assert takes_tensor_cores(x, wg, wu, off)

    def moved(t, around):
        buf = torch.full((t.numel() + 16,), around, device=cuda)
        view = buf[shift:shift + t.numel()].view(t.shape)
        return buf, view.copy_(t)

    h, gu = forward(x, wg, wu, off)
    hb, h2 = moved(torch.zeros_like(h), 9.0)
    gb, gu2 = moved(torch.zeros_like(gu), 9.0)
    nan = float("nan")
    rr.grouped_gated_gemm(moved(x, nan)[1], moved(wg, nan)[1], moved(wu, nan)[1], off, h2,
                          gate_up=gu2, workspace=workspace(x, wg))
    assert torch.equal(h, h2) and torch.equal(gu, gu2)
    for buf, t in ((hb, h), (gb, gu)):
        assert bool((buf[:shift] == 9.0).all()) and bool((buf[shift + t.numel():] == 9.0).all())


# (experts, K, N, the most rows of the plain form): N a multiple of 4 and not.
@pytest.mark.parametrize("edge", [(3, 128, 128, 756), (6, 520, 264, 400), (5, 130, 129, 368),
                                  (7, 333, 259, 208)], ids=str)
def test_forms_meet(cuda, edge):
    e, k, n, most = edge
    for rows, engine in ((most, False), (most + 1, True)):
        counts = np.random.default_rng(rows).multinomial(rows, [1 / e] * e)
        x, wg, wu, off, _ = make(counts, 0, k, n, FP32, cuda, seed=81)
        assert takes_tensor_cores(x, wg, wu, off) == engine
        h, gu = forward(x, wg, wu, off)
        g, u, want = gated(x, wg, wu, off)
        assert normwise(h, want) < 2.0 ** -19
        assert normwise(gu, torch.cat((g, u), 1)) < 2.0 ** -20
