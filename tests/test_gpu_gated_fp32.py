"""rr_grouped_gated_gemm and its backward pass in FP32 where the tensor-core form
runs."""
from __future__ import annotations

import pytest
import torch

import raggedroute_b200 as rr
from expert_block_reference import offsets_of
from test_gpu_gated import backward, forward, no_device_error

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
