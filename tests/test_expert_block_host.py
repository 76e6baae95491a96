"""What the expert-block operators refuse, and their workspace sizes (no GPU):
every refusal comes before anything is launched or read."""
from __future__ import annotations

import ctypes

import pytest
import torch

from raggedroute_b200 import RaggedRouteError, StatusCode
from raggedroute_b200 import expert_block as block
from raggedroute_b200._lib import Context, RRContext

A = 1 << 20  # stand-ins for device addresses, far apart; never read here
BUF = [A + (i << 32) for i in range(20)]


def ctx(workspace=0, size=0):
    c = Context(workspace=workspace, workspace_bytes=size)
    return ctypes.pointer(c.as_c())


def code(status):
    return StatusCode(status.code)


def gated(lib, x=BUF[0], wg=BUF[1], wu=BUF[2], off=BUF[3], h=BUF[4], gu=None, rows=64, e=4, k=64,
          n=64, act=0, dtype=2, c=None):
    return code(lib.rr_grouped_gated_gemm(x, wg, wu, off, h, gu, rows, e, k, n, act, dtype,
                                          c or ctx()))


def gated_back(lib, dx=BUF[6], dg=BUF[7], du=BUF[8], gu=BUF[5], dh=BUF[4], rows=64, e=4, k=64,
               n=64, act=0, dtype=2, c=None):
    return code(lib.rr_grouped_gated_gemm_backward(BUF[0], BUF[1], BUF[2], BUF[3], gu, dh, dx, dg,
                                                   du, rows, e, k, n, act, dtype, c or ctx()))


def test_gated_refusals(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT
    for kw in (dict(rows=-1), dict(e=0), dict(e=1025), dict(k=0), dict(n=0), dict(act=3),
               dict(act=-1), dict(x=None), dict(wg=None), dict(wu=None), dict(off=None),
               dict(h=None), dict(x=BUF[0] + 2), dict(wg=BUF[1] + 8), dict(h=BUF[4] + 2),
               dict(gu=BUF[5] + 4), dict(off=BUF[3] + 2), dict(x=BUF[0] + 1, k=63),
               dict(h=BUF[0]), dict(h=BUF[1] + 16), dict(gu=BUF[4])):
        assert gated(lib, **kw) == bad, kw
    for dtype in (1, 3, -1, 99):
        assert gated(lib, dtype=dtype) == StatusCode.UNSUPPORTED_DATA_TYPE
    null = lib.rr_grouped_gated_gemm(*BUF[:5], None, 64, 4, 64, 64, 0, 2, None)
    assert code(null) == bad
    # FP32 needs its workspace above the few-row form; so do odd rows.
    for kw in (dict(dtype=0, rows=4096), dict(k=63, rows=4096)):
        assert gated(lib, **kw) == StatusCode.INSUFFICIENT_WORKSPACE, kw
    size = lib.rr_grouped_gated_gemm_workspace_size(4096, 4, 64, 64, 0)
    assert gated(lib, dtype=0, rows=4096, c=ctx(BUF[9], size - 1)) == \
        StatusCode.INSUFFICIENT_WORKSPACE
    assert gated(lib, dtype=0, rows=4096, c=ctx(BUF[9] + 16, size)) == bad
    assert gated(lib, rows=0, x=None, h=None) == StatusCode.SUCCESS


def test_gated_backward_refusals(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT
    for kw in (dict(dg=None), dict(du=None), dict(dx=None, dg=None, du=None), dict(gu=None),
               dict(dh=None), dict(dx=BUF[0]), dict(dx=BUF[4]), dict(dg=BUF[8]), dict(dg=BUF[1]),
               dict(dx=BUF[6] + 2), dict(act=7), dict(k=0), dict(rows=-5)):
        assert gated_back(lib, **kw) == bad, kw
    assert gated_back(lib, dtype=1) == StatusCode.UNSUPPORTED_DATA_TYPE
    assert gated_back(lib) == StatusCode.INSUFFICIENT_WORKSPACE
    assert gated_back(lib, rows=0, dg=None, du=None) == StatusCode.SUCCESS


def test_gated_workspace(rrlib):
    size = rrlib.lib().rr_grouped_gated_gemm_workspace_size
    back = rrlib.lib().rr_grouped_gated_gemm_backward_workspace_size
    assert size(4096, 8, 64, 64, 2) == 0           # read in place
    assert size(4, 8, 63, 63, 2) == 0              # few rows: read in place
    assert size(4096, 8, 63, 64, 2) == 4096 * 64 * 2
    assert size(4096, 8, 64, 63, 2) == 2 * 8 * 64 * 64 * 2
    assert size(4096, 8, 64, 64, 0) == 6 * (4096 * 64 + 2 * 8 * 64 * 64)
    assert back(4096, 8, 64, 64, 2) == 2 * 4096 * 64 * 2
    assert back(4096, 8, 64, 64, 0) == 6 * (3 * 4096 * 64 + 2 * 8 * 64 * 64)
    assert back(4, 8, 64, 64, 2) == 2 * 4 * 64 * 4   # few rows: dg and du in FP32
    assert back(64, 8, 64, 64, 0) == 2 * 64 * 64 * 4
    # Rows scarce among the experts keep a second part of dg and du.
    assert back(256, 8, 64, 64, 2) == 2 * 2 * 256 * 64 * 2
    # Past 32 bits: 131072 rows of the 128-expert layer in FP32.
    assert size(131072, 128, 4096, 1408, 0) == 6 * (131072 * 4096 + 2 * 128 * 4096 * 1408)
    for bad in ((-1, 8, 64, 64, 0), (1, 0, 64, 64, 0), (1, 8, 0, 64, 0), (1, 8, 64, 64, 1)):
        assert size(*bad) == 0 and back(*bad) == 0


def test_int8_refusals(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT

    def rows(x=BUF[0], xq=BUF[1], s=BUF[2], r=4, k=64, dtype=2):
        return code(lib.rr_quantize_rows_int8(x, xq, s, r, k, dtype, ctx()))

    for kw in (dict(x=None), dict(xq=None), dict(s=None), dict(xq=BUF[1] + 8), dict(x=BUF[0] + 1),
               dict(r=-1), dict(k=0), dict(k=131073), dict(xq=BUF[0]), dict(s=BUF[1] + 16)):
        assert rows(**kw) == bad, kw
    assert rows(dtype=1) == StatusCode.UNSUPPORTED_DATA_TYPE
    assert rows(r=0, x=None) == StatusCode.SUCCESS

    def weights(w=BUF[0], wq=BUF[1], s=BUF[2], e=4, k=64, n=8, dtype=0):
        return code(lib.rr_quantize_expert_weights_int8(w, wq, s, e, k, n, dtype, ctx()))

    for kw in (dict(w=None), dict(wq=None), dict(s=None), dict(wq=BUF[1] + 4), dict(e=0),
               dict(e=1025), dict(k=0), dict(k=131073), dict(n=0), dict(wq=BUF[0])):
        assert weights(**kw) == bad, kw
    assert weights(dtype=5) == StatusCode.UNSUPPORTED_DATA_TYPE

    def product(xq=BUF[0], xs=BUF[1], wq=BUF[2], ws=BUF[3], off=BUF[4], y=BUF[5], r=64, e=4, k=64,
                n=64, dtype=2):
        return code(lib.rr_grouped_gemm_int8(xq, xs, wq, ws, off, y, r, e, k, n, dtype, ctx()))

    for kw in (dict(xq=None), dict(xs=None), dict(wq=None), dict(ws=None), dict(off=None),
               dict(y=None), dict(xq=BUF[0] + 8), dict(wq=BUF[2] + 1), dict(y=BUF[5] + 2),
               dict(y=BUF[0]), dict(r=-1), dict(e=0), dict(e=2000), dict(k=0), dict(k=131073),
               dict(n=0), dict(xs=BUF[1] + 2)):
        assert product(**kw) == bad, kw
    assert product(dtype=1) == StatusCode.UNSUPPORTED_DATA_TYPE
    assert product(r=0) == StatusCode.SUCCESS
    assert [lib.rr_int8_row_stride(k) for k in (-1, 0, 1, 16, 17, 131072, 131073)] == \
        [0, 0, 16, 16, 32, 131072, 0]


def test_norm_refusals(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT

    def norm(yp=BUF[0], pos=BUF[1], w=BUF[2], res=BUF[3], post=BUF[4], gate=BUF[5], pre=BUF[6],
             out=BUF[7], normed=BUF[8], inv=BUF[9], eps=1e-6, t=8, k=2, n=64, dtype=2):
        return code(lib.rr_unpermute_norm(yp, pos, w, res, post, gate, pre, out, normed, inv, eps,
                                          1.0, t, k, n, dtype, ctx()))

    for kw in (dict(yp=None), dict(pos=None), dict(w=None), dict(res=None), dict(out=None),
               dict(pre=None), dict(normed=None), dict(eps=-1.0), dict(eps=float("nan")),
               dict(t=-1), dict(k=0), dict(k=65), dict(n=0), dict(n=16385), dict(t=2 ** 30, k=2),
               dict(out=BUF[0]), dict(out=BUF[3] + 16), dict(normed=BUF[7]), dict(normed=BUF[3]),
               dict(inv=BUF[8]), dict(post=BUF[4] + 2), dict(res=BUF[3] + 1)):
        assert norm(**kw) == bad, kw
    assert norm(dtype=1) == StatusCode.UNSUPPORTED_DATA_TYPE
    assert norm(t=0, yp=None) == StatusCode.SUCCESS

    def back(yp=BUF[0], post=BUF[4], gate=BUF[5], pre=BUF[6], inv=BUF[7], dro=BUF[8], dn=BUF[9],
             dres=BUF[10], dyp=BUF[11], dw=BUF[12], dpost=BUF[13], dgate=BUF[14], dpre=BUF[15],
             t=8, k=2, n=64, dtype=2):
        return code(lib.rr_unpermute_norm_backward(yp, BUF[1], BUF[2], BUF[3], post, gate, pre,
                                                   inv, dro, dn, dres, dyp, dw, dpost, dgate,
                                                   dpre, 1.0, t, k, n, dtype, ctx()))

    for kw in (dict(yp=None), dict(inv=None), dict(dres=None), dict(dyp=None), dict(dw=None),
               dict(post=None), dict(gate=None), dict(pre=None), dict(pre=None, dpre=None),
               dict(dyp=BUF[0]), dict(dyp=BUF[8]), dict(dres=BUF[9]), dict(dres=BUF[8] + 16),
               dict(dgate=BUF[13]), dict(dw=BUF[2]), dict(t=-1), dict(n=16385), dict(k=0)):
        assert back(**kw) == bad, kw
    assert back() == StatusCode.INSUFFICIENT_WORKSPACE
    assert back(dtype=4) == StatusCode.UNSUPPORTED_DATA_TYPE
    size = lib.rr_unpermute_norm_backward_workspace_size
    assert size(0, 64) == 0 and size(-1, 64) == 0 and size(8, 16385) == 0
    assert size(1, 64) == 12 * 64 and size(10 ** 6, 4096) <= 12 * 4096 * 148 * 16


def test_python_refusals(rrlib):
    """Types, shapes, strides and devices, before the library is called."""
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError, match="CUDA"):
        block.quantize_rows_int8(x, torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4))
    for dtype in (torch.float16, torch.float64, torch.int32):
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            block.quantize_rows_int8(x.to(dtype), torch.zeros(4, 16, dtype=torch.int8),
                                     torch.zeros(4))
    with pytest.raises(ValueError, match="131072"):
        block.int8_row_stride(131073)
    with pytest.raises(TypeError):
        block.grouped_gated_gemm_workspace_size(4, 4, 16, 16, torch.float16)
    w = torch.zeros(2, 16, 8)
    with pytest.raises(ValueError, match="CUDA"):
        block.grouped_gated_gemm(x, w, w, torch.zeros(3, dtype=torch.int32), torch.zeros(4, 8))
    with pytest.raises(ValueError, match="activation"):
        block._activation("swish2")
    dev = x.device
    with pytest.raises(ValueError, match="shape"):
        block._expect(x, (4, 15), torch.float32, dev, "x")
    with pytest.raises(ValueError, match="contiguous"):
        block._expect(x.t(), (16, 4), torch.float32, dev, "x")
    with pytest.raises(TypeError, match="float32"):
        block._expect(x.double(), (4, 16), torch.float32, dev, "x")
    with pytest.raises(ValueError, match="must be on"):
        block._expect(x, (4, 16), torch.float32, torch.device("cuda", 0), "x")


def test_error_names_the_operator(rrlib):
    with pytest.raises(RaggedRouteError, match="grouped_gated_gemm: INVALID_ARGUMENT"):
        status = rrlib.lib().rr_grouped_gated_gemm(None, None, None, None, None, None, 4, 4, 4, 4,
                                                   0, 2, ctypes.pointer(RRContext()))
        from raggedroute_b200._lib import check
        check(status, "grouped_gated_gemm")


def test_workspace_that_touches_a_buffer(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT
    size = lib.rr_grouped_gated_gemm_workspace_size(4096, 4, 64, 64, 0)
    for buf in (BUF[0], BUF[1], BUF[4] + 256):  # x, gate weights, h
        assert gated(lib, dtype=0, rows=4096, c=ctx(buf, size)) == bad, hex(buf)
    size = lib.rr_grouped_gated_gemm_backward_workspace_size(64, 4, 64, 64, 2)
    for buf in (BUF[0], BUF[5], BUF[7], BUF[6] - size + 256):  # x, gate_up, dWg, in front of dx
        assert gated_back(lib, c=ctx(buf, size)) == bad, hex(buf)
    size = lib.rr_unpermute_norm_backward_workspace_size(8, 64)
    for buf in (BUF[0], BUF[3], BUF[8], BUF[11], BUF[15]):
        assert code(lib.rr_unpermute_norm_backward(
            *BUF[:16], 1.0, 8, 2, 64, 2, ctx(buf, size))) == bad, hex(buf)


def test_dimensions_past_an_int(rrlib):
    """A long dimension is refused, not cut to 32 bits."""
    x = torch.empty(2 ** 31, 1, device="meta", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="longer than"):
        block.quantize_rows_int8(x, x, x)
    w = torch.empty(2, 1, 2 ** 31, device="meta")
    with pytest.raises(ValueError, match="longer than"):
        block.quantize_expert_weights_int8(w, w, w)


def test_sizes_past_the_index_range(rrlib):
    lib = rrlib.lib()
    bad = StatusCode.INVALID_ARGUMENT
    assert gated(lib, k=2 ** 30 + 8) == bad and gated(lib, n=2 ** 29 + 8) == bad
    assert gated_back(lib, k=2 ** 30 + 8) == bad and gated_back(lib, n=2 ** 29 + 8) == bad
    assert lib.rr_grouped_gated_gemm_workspace_size(64, 4, 2 ** 30 + 8, 64, 0) == 0
    assert code(lib.rr_grouped_gemm_int8(*BUF[:6], 64, 4, 64, 2 ** 30 + 16, 2, ctx())) == bad
    assert code(lib.rr_quantize_expert_weights_int8(*BUF[:3], 4, 64, 2 ** 30 + 16, 2, ctx())) == bad
