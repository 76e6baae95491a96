"""rr_quantize_rows_int8, rr_quantize_expert_weights_int8 and
rr_grouped_gemm_int8.

The quantised values are compared for equality with the definition evaluated in
float32 on the host (IEEE division, product and rounding); the product's sum is
exact, and its scaling adds at most three FP32 roundings and the output's one.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_b200 as rr
from expert_block_reference import half_step, offsets_of, random

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def quantized(x: torch.Tensor, axis: int):
    """(q, scale) of the definition, in float32 on the host."""
    v = x.float().cpu().numpy()
    top = np.abs(v).max(axis=axis, keepdims=True)
    top = np.where(top < np.float32(2.0 ** -120), np.float32(0), top)
    with np.errstate(divide="ignore", invalid="ignore"):
        inverse = np.where(top > 0, np.float32(127) / top, np.float32(0)).astype(np.float32)
        q = np.rint(v * inverse)
    return q.astype(np.int32), (top / np.float32(127)).squeeze(axis)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 16), (5, 33), (70, 64), (17, 1001),
                                         (4, 4096), (3, 9000), (2, 20007)])
def test_quantize_rows(cuda, rows, hidden, dtype):
    x = random((rows, hidden), 1, cuda, dtype, 3.0)
    x[0] = 0
    if rows > 2:
        x[1] = x[1] * 2.0 ** -122  # wholly below the smallest magnitude that counts
        x[2] = x[2] * 1e30
    stride = rr.int8_row_stride(hidden)
    xq = torch.full((rows, stride), 99, dtype=torch.int8, device=cuda)
    scale = torch.full((rows,), 5.0, device=cuda)
    rr.quantize_rows_int8(x, xq, scale)
    q, s = quantized(x, 1)
    assert np.array_equal(xq[:, :hidden].cpu().numpy(), q)
    assert not xq[:, hidden:].any()
    assert np.array_equal(scale.cpu().numpy(), s)
    assert int(xq.abs().max()) <= 127


def test_quantize_rows_not_finite(cuda):
    x = random((4, 64), 2, cuda)
    x[1, 5] = float("inf")
    x[2, 63] = float("nan")
    xq = torch.zeros(4, 64, dtype=torch.int8, device=cuda)
    scale = torch.zeros(4, device=cuda)
    rr.quantize_rows_int8(x, xq, scale)
    assert torch.isfinite(scale[0]) and torch.isinf(scale[1]) and torch.isnan(scale[2])
    w = random((1, 64, 40), 3, cuda)
    wq = torch.zeros(1, 40, 64, dtype=torch.int8, device=cuda)
    ws = torch.zeros(1, 40, device=cuda)
    rr.quantize_expert_weights_int8(w, wq, ws)
    for reps in (1, 20):  # the few-row form and the tensor-core form
        y = torch.zeros(4 * reps, 40, device=cuda)
        rr.grouped_gemm_int8(xq.repeat(reps, 1), scale.repeat(reps), wq, ws,
                             offsets_of([4 * reps], cuda), y)
        assert torch.isnan(y[1::4]).all() and torch.isnan(y[2::4]).all()
        assert torch.isfinite(y[0::4]).all() and torch.isfinite(y[3::4]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("experts,hidden,output", [(1, 1, 1), (3, 16, 8), (2, 33, 70),
                                                   (5, 200, 64), (2, 1001, 131)])
def test_quantize_weights(cuda, experts, hidden, output, dtype):
    w = random((experts, hidden, output), 4, cuda, dtype, 0.3)
    w[0, :, 0] = 0
    stride = rr.int8_row_stride(hidden)
    wq = torch.full((experts, output, stride), 99, dtype=torch.int8, device=cuda)
    ws = torch.full((experts, output), 5.0, device=cuda)
    rr.quantize_expert_weights_int8(w, wq, ws)
    q, s = quantized(w, 1)
    assert np.array_equal(wq[:, :, :hidden].cpu().numpy(), q.transpose(0, 2, 1))
    assert not wq[:, :, hidden:].any()
    assert np.array_equal(ws.cpu().numpy(), s)


def product(xq, xs, wq, ws, off):
    out = torch.zeros(xq.shape[0], wq.shape[1], dtype=torch.float64, device=xq.device)
    o = off.tolist()
    for e, (a, b) in enumerate(zip(o, o[1:])):
        out[a:b] = (xq[a:b].double() @ wq[e].double().T) * xs[a:b, None].double() * ws[e].double()
    return out


def operands(rows, experts, hidden, output, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    stride = rr.int8_row_stride(hidden)

    def ints(*shape):
        t = torch.randint(-127, 128, shape, generator=g, device=device, dtype=torch.int8)
        t[..., hidden:] = 0
        return t

    return (ints(rows, stride), torch.rand(rows, generator=g, device=device) + 0.1,
            ints(experts, output, stride),
            torch.rand(experts, output, generator=g, device=device) + 0.1)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("counts,behind,hidden,output", [
    ([1], 0, 1, 1),
    ([0, 2, 0, 1], 1, 16, 8),
    ([7, 0, 9, 3], 2, 100, 33),
    ([32], 0, 512, 64),
    ([33], 0, 512, 64),
    ([64, 1, 63], 4, 130, 129),
    ([0, 257, 129, 0], 0, 384, 256),
    ([300, 500], 9, 1030, 515),
    ([20] * 70, 0, 64, 40),
    ([90], 0, 20000, 24),
    ([700, 0, 1100, 257, 513, 130, 385, 1], 3, 4100, 6700),  # two row blocks share a tile
], ids=str)
def test_product(cuda, counts, behind, hidden, output, dtype):
    rows = int(np.sum(counts)) + behind
    xq, xs, wq, ws = operands(rows, len(counts), hidden, output, cuda)
    off = offsets_of(counts, cuda)
    y = torch.full((rows, output), 777.0, dtype=dtype, device=cuda)
    rr.grouped_gemm_int8(xq, xs, wq, ws, off, y)
    n = rows - behind
    want = product(xq, xs, wq, ws, off)[:n]
    tol = (half_step(dtype) + 4 * 2.0 ** -24) * want.abs()
    assert bool(((y[:n].double() - want).abs() <= tol).all())
    assert bool((y[n:] == 777.0).all())
    again = torch.full_like(y, 777.0)
    rr.grouped_gemm_int8(xq, xs, wq, ws, off, again)
    assert torch.equal(y, again)


def test_largest_sums(cuda):
    """All products at +-127^2 over the longest row: no 32-bit overflow."""
    hidden = 131072
    xq = torch.full((40, hidden), 127, dtype=torch.int8, device=cuda)
    wq = torch.full((1, 3, hidden), 127, dtype=torch.int8, device=cuda)
    wq[0, 1] = -127
    one = torch.ones(40, device=cuda)
    for rows in (2, 40):
        y = torch.zeros(rows, 3, device=cuda)
        rr.grouped_gemm_int8(xq[:rows], one[:rows], wq, torch.ones(1, 3, device=cuda),
                             offsets_of([rows], cuda), y)
        total = float(127 * 127 * hidden)
        assert torch.equal(y, torch.tensor([total, -total, total], device=cuda).expand(rows, 3))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_whole_path_is_near_the_product(cuda, dtype):
    """Quantised rows times quantised weights, against x . W in float64: each
    operand is off by at most half a step of its scale."""
    rows, experts, k, n = 300, 3, 256, 96
    x, w = random((rows, k), 5, cuda, dtype), random((experts, k, n), 6, cuda, dtype, 0.1)
    off = offsets_of([100, 0, 200], cuda)
    xq = torch.empty(rows, k, dtype=torch.int8, device=cuda)
    wq = torch.empty(experts, n, k, dtype=torch.int8, device=cuda)
    xs, ws = torch.empty(rows, device=cuda), torch.empty(experts, n, device=cuda)
    y = torch.empty(rows, n, dtype=dtype, device=cuda)
    rr.quantize_rows_int8(x, xq, xs)
    rr.quantize_expert_weights_int8(w, wq, ws)
    rr.grouped_gemm_int8(xq, xs, wq, ws, off, y)
    o = off.tolist()
    for e, (a, b) in enumerate(zip(o, o[1:])):
        xe, we = x[a:b].double(), w[e].double()
        ex, ew = 0.5001 * xs[a:b, None].double(), 0.5001 * ws[e][None].double()
        tol = ex * we.abs().sum(0) + ew * xe.abs().sum(1, keepdim=True) + k * ex * ew
        want = xe @ we
        tol = tol * (1 + half_step(dtype)) + (half_step(dtype) + 2.0 ** -21) * want.abs()
        assert bool(((y[a:b].double() - want).abs() <= tol).all())


def test_replay(cuda):
    xq, xs, wq, ws = operands(100, 4, 96, 56, cuda, 7)
    x = random((100, 96), 8, cuda, BF16)
    off = offsets_of([10, 50, 0, 40], cuda)
    y = torch.zeros(100, 56, dtype=BF16, device=cuda)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step(ctx):
        rr.quantize_rows_int8(x, xq, xs, ctx=ctx)
        rr.grouped_gemm_int8(xq, xs, wq, ws, off, y, ctx=ctx)

    graph = rr.Graph.capture(step, s)
    for seed, counts in ((8, [10, 50, 0, 40]), (9, [0, 0, 100, 0])):
        x.copy_(random((100, 96), seed, cuda, BF16))
        off.copy_(offsets_of(counts, cuda))
        torch.cuda.synchronize()
        graph.launch(s)
        s.synchronize()
        got = y.clone()
        step(None)
        torch.cuda.synchronize()
        assert torch.equal(got, y)
