"""Expert-block operators over the C ABI: the gated expert projection and its
backward pass, the 8-bit integer grouped product, and the weighted combine with
the norms, gate and residual at a block's end, with its backward pass.

As in raggedroute_b200.ops, functions take contiguous CUDA tensors and
caller-owned outputs, check types and shapes on the host and call the matching
``rr_*`` entry point on the current torch stream (or ``ctx.stream``). float32
and bfloat16 are accepted; sizes are read from the tensors. A call runs on the
device of its tensors. No reference counterpart.

The operators of a forward or backward pass go through the compiled binding
(csrc/python/block_calls.cpp), which makes the same checks; where one fails, or
``ctx`` is given, or the tensors are on another device than the current one, the
Python below makes the call and names what is wrong.
"""
from __future__ import annotations

import ctypes

import torch

from raggedroute_b200._lib import (Context, RaggedRouteError, RRContext, StatusCode, check, lib)
from raggedroute_b200.ops import _need

_MAX_SIZE = 2**31 - 1  # the entry points take sizes as int
_DTYPES = {torch.float32: 0, torch.bfloat16: 2}
ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "relu": 2}


_calls = None


def _load():
    """The compiled binding (raises if it is missing)."""
    global _calls
    lib()
    try:
        from raggedroute_b200 import _block_calls
    except ImportError as e:
        raise RaggedRouteError(int(StatusCode.CUDA_ERROR), 0, f"{e}; run "
                               "`python -m raggedroute_b200.build`", "load") from e
    _block_calls.set_error(RaggedRouteError)
    _calls = _block_calls
    return _calls


def _dtype(dtype: torch.dtype, name: str) -> int:
    if dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {dtype}")
    return _DTYPES[dtype]


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def _refuse(t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device,
            name: str) -> None:
    _need(t, dtype, name)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be on {device}, got {t.device}")


def _expect(t: torch.Tensor | None, shape: tuple, dtype: torch.dtype, device: torch.device,
            name: str) -> int | None:
    """The address of `t`, a contiguous tensor of this shape, type and device;
    None passes as a null pointer."""
    if t is None:
        return None
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        _refuse(t, shape, dtype, device, name)
    return t.data_ptr() or None


def _rank(t: torch.Tensor, dims: int, name: str) -> None:
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {t.dim()}")
    if t.numel() > _MAX_SIZE and max(t.shape) > _MAX_SIZE:
        raise ValueError(f"{name}: no dimension may be longer than {_MAX_SIZE}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor, got {t.device}")


def _call(fn, name: str, device: torch.device, ctx: Context | None,
          workspace: torch.Tensor | None, *args) -> None:
    """fn(*args, context) with `device` current, on its current stream unless
    ctx names one."""
    if workspace is not None and (workspace.device != device or not workspace.is_contiguous()):
        raise ValueError(f"workspace must be a contiguous tensor on {device}")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(fn, name, device, ctx, workspace, *args)
    if ctx is not None:
        c = ctx.as_c()
        if not c.stream:
            c.stream = torch.cuda.current_stream().cuda_stream
    else:
        c = RRContext(torch._C._cuda_getCurrentRawStream(device.index))
    if workspace is not None:
        c.workspace = workspace.data_ptr()
        c.workspace_bytes = workspace.numel() * workspace.element_size()
    status = fn(*args, ctypes.byref(c))
    if status.code != 0:
        check(status, name)


# ---- gated projection ------------------------------------------------------------

def grouped_gated_gemm_workspace_size(route_pairs: int, experts: int, hidden: int, output: int,
                                      dtype: torch.dtype, backward: bool = False) -> int:
    """Workspace bytes of grouped_gated_gemm, or with `backward` of it and
    grouped_gated_gemm_backward."""
    sizes = (route_pairs, experts, hidden, output, _dtype(dtype, "dtype"))
    size = int(lib().rr_grouped_gated_gemm_workspace_size(*sizes))
    if backward:
        size = max(size, int(lib().rr_grouped_gated_gemm_backward_workspace_size(*sizes)))
    return size


def _gated_inputs(x: torch.Tensor, gate_weights: torch.Tensor, up_weights: torch.Tensor,
                  offsets: torch.Tensor):
    """((rows, experts, hidden, output), the four addresses)."""
    _rank(x, 2, "x_permuted")
    _rank(gate_weights, 3, "gate_weights")
    rows, hidden = x.shape
    experts, _, output = w_shape = gate_weights.shape
    if w_shape[1] != hidden:
        raise ValueError(f"gate_weights must be [E, {hidden}, N], got {tuple(w_shape)}")
    dtype, device = x.dtype, x.device
    return (rows, experts, hidden, output), (
        _expect(x, x.shape, dtype, device, "x_permuted"),
        _expect(gate_weights, w_shape, dtype, device, "gate_weights"),
        _expect(up_weights, w_shape, dtype, device, "up_weights"),
        _expect(offsets, (experts + 1,), torch.int32, device, "offsets"))


def grouped_gated_gemm(x_permuted: torch.Tensor, gate_weights: torch.Tensor,
                       up_weights: torch.Tensor, offsets: torch.Tensor, h: torch.Tensor,
                       gate_up: torch.Tensor | None = None, activation: str = "silu",
                       workspace: torch.Tensor | None = None,
                       ctx: Context | None = None) -> torch.Tensor:
    """h[r] = act(x[r] . Wg[e]) * (x[r] . Wu[e]) for the rows of each expert's
    segment (rr_grouped_gated_gemm). x_permuted [R, K], gate_weights and
    up_weights [E, K, N], h [R, N]; gate_up (float32 [R, 2N]) receives both
    products for the backward pass. activation: silu, gelu_tanh or relu.
    workspace from grouped_gated_gemm_workspace_size."""
    if ctx is None and activation in ACTIVATIONS and (_calls or _load()).grouped_gated_gemm(
            x_permuted, gate_weights, up_weights, offsets, h, gate_up, ACTIVATIONS[activation],
            workspace):
        return h
    dtype, act = _dtype(x_permuted.dtype, "x_permuted"), _activation(activation)
    sizes, inputs = _gated_inputs(x_permuted, gate_weights, up_weights, offsets)
    rows, _, _, output = sizes
    device = x_permuted.device
    _call(lib().rr_grouped_gated_gemm, "grouped_gated_gemm", device, ctx, workspace, *inputs,
          _expect(h, (rows, output), x_permuted.dtype, device, "h"),
          _expect(gate_up, (rows, 2 * output), torch.float32, device, "gate_up"), *sizes, act,
          dtype)
    return h


def grouped_gated_gemm_backward(x_permuted: torch.Tensor, gate_weights: torch.Tensor,
                                up_weights: torch.Tensor, offsets: torch.Tensor,
                                gate_up: torch.Tensor, dh: torch.Tensor,
                                dx: torch.Tensor | None, d_gate_weights: torch.Tensor | None,
                                d_up_weights: torch.Tensor | None, activation: str = "silu",
                                workspace: torch.Tensor | None = None,
                                ctx: Context | None = None) -> None:
    """Gradients of grouped_gated_gemm from dh [R, N] and the saved gate_up
    (rr_grouped_gated_gemm_backward). dx [R, K] may be None, or both weight
    gradients [E, K, N]. workspace from
    grouped_gated_gemm_workspace_size(..., backward=True)."""
    if ctx is None and activation in ACTIVATIONS and (
            _calls or _load()).grouped_gated_gemm_backward(
                x_permuted, gate_weights, up_weights, offsets, gate_up, dh, dx, d_gate_weights,
                d_up_weights, ACTIVATIONS[activation], workspace):
        return
    dtype, act = _dtype(x_permuted.dtype, "x_permuted"), _activation(activation)
    sizes, inputs = _gated_inputs(x_permuted, gate_weights, up_weights, offsets)
    rows, experts, hidden, output = sizes
    t, device, weights = x_permuted.dtype, x_permuted.device, (experts, hidden, output)
    _call(lib().rr_grouped_gated_gemm_backward, "grouped_gated_gemm_backward", device, ctx,
          workspace, *inputs,
          _expect(gate_up, (rows, 2 * output), torch.float32, device, "gate_up"),
          _expect(dh, (rows, output), t, device, "dh"),
          _expect(dx, (rows, hidden), t, device, "dx"),
          _expect(d_gate_weights, weights, t, device, "d_gate_weights"),
          _expect(d_up_weights, weights, t, device, "d_up_weights"), *sizes, act, dtype)


# ---- 8-bit integers ----------------------------------------------------------------

def int8_row_stride(hidden: int) -> int:
    """Bytes of a quantised row: hidden rounded up to 16."""
    stride = int(lib().rr_int8_row_stride(hidden))
    if stride == 0:
        raise ValueError(f"hidden must be in [1, 131072], got {hidden}")
    return stride


def quantize_rows_int8(x: torch.Tensor, xq: torch.Tensor, x_scale: torch.Tensor,
                       ctx: Context | None = None) -> None:
    """Rows of x [R, K] in 8-bit integers with one scale each
    (rr_quantize_rows_int8): xq int8 [R, int8_row_stride(K)], x_scale float32
    [R]; x is close to xq * x_scale."""
    if ctx is None and (_calls or _load()).quantize_rows_int8(x, xq, x_scale):
        return
    dtype = _dtype(x.dtype, "x")
    _rank(x, 2, "x")
    rows, hidden = x.shape
    device = x.device
    _call(lib().rr_quantize_rows_int8, "quantize_rows_int8", device, ctx, None,
          _expect(x, x.shape, x.dtype, device, "x"),
          _expect(xq, (rows, int8_row_stride(hidden)), torch.int8, device, "xq"),
          _expect(x_scale, (rows,), torch.float32, device, "x_scale"), rows, hidden, dtype)


def quantize_expert_weights_int8(expert_weights: torch.Tensor, wq: torch.Tensor,
                                 w_scale: torch.Tensor, ctx: Context | None = None) -> None:
    """Expert weights [E, K, N] in 8-bit integers with one scale per output
    channel (rr_quantize_expert_weights_int8): wq int8 [E, N,
    int8_row_stride(K)], w_scale float32 [E, N]. Done once per weight set."""
    dtype = _dtype(expert_weights.dtype, "expert_weights")
    _rank(expert_weights, 3, "expert_weights")
    experts, hidden, output = expert_weights.shape
    device = expert_weights.device
    _call(lib().rr_quantize_expert_weights_int8, "quantize_expert_weights_int8", device, ctx, None,
          _expect(expert_weights, expert_weights.shape, expert_weights.dtype, device,
                  "expert_weights"),
          _expect(wq, (experts, output, int8_row_stride(hidden)), torch.int8, device, "wq"),
          _expect(w_scale, (experts, output), torch.float32, device, "w_scale"), experts, hidden,
          output, dtype)


def grouped_gemm_int8(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor,
                      w_scale: torch.Tensor, offsets: torch.Tensor, y_permuted: torch.Tensor,
                      ctx: Context | None = None) -> torch.Tensor:
    """y[r] = (xq[r] . wq[e]^T) * x_scale[r] * w_scale[e] for the rows of each
    expert's segment (rr_grouped_gemm_int8), from quantize_rows_int8 and
    quantize_expert_weights_int8; y_permuted [R, N] float32 or bfloat16."""
    if ctx is None and (_calls or _load()).grouped_gemm_int8(xq, x_scale, wq, w_scale, offsets,
                                                             y_permuted):
        return y_permuted
    dtype = _dtype(y_permuted.dtype, "y_permuted")
    _rank(xq, 2, "xq")
    _rank(wq, 3, "wq")
    rows, stride = xq.shape
    experts, output, _ = wq.shape
    device = xq.device
    if int8_row_stride(stride) != stride:
        raise ValueError(f"xq rows must be int8_row_stride(K) long, got {stride}")
    _call(lib().rr_grouped_gemm_int8, "grouped_gemm_int8", device, ctx, None,
          _expect(xq, xq.shape, torch.int8, device, "xq"),
          _expect(x_scale, (rows,), torch.float32, device, "x_scale"),
          _expect(wq, (experts, output, stride), torch.int8, device, "wq"),
          _expect(w_scale, (experts, output), torch.float32, device, "w_scale"),
          _expect(offsets, (experts + 1,), torch.int32, device, "offsets"),
          _expect(y_permuted, (rows, output), y_permuted.dtype, device, "y_permuted"), rows,
          experts, stride, output, dtype)
    return y_permuted


# ---- combine, norms, gate, residual --------------------------------------------------

def _norm_inputs(y_permuted, route_pos, route_weights, residual, post_gamma, gate, pre_gamma):
    """((tokens, top_k, output), the seven addresses)."""
    _rank(residual, 2, "residual")
    _rank(route_pos, 2, "route_pos")
    tokens, output = residual.shape
    top_k = route_pos.shape[1]
    t, device, f32 = residual.dtype, residual.device, torch.float32
    return (tokens, top_k, output), (
        _expect(y_permuted, (tokens * top_k, output), t, device, "y_permuted"),
        _expect(route_pos, (tokens, top_k), torch.int32, device, "route_pos"),
        _expect(route_weights, (tokens, top_k), f32, device, "route_weights"),
        _expect(residual, residual.shape, t, device, "residual"),
        _expect(post_gamma, (output,), f32, device, "post_gamma"),
        _expect(gate, (output,), f32, device, "gate"),
        _expect(pre_gamma, (output,), f32, device, "pre_gamma"))


def unpermute_norm(y_permuted: torch.Tensor, route_pos: torch.Tensor,
                   route_weights: torch.Tensor, residual: torch.Tensor,
                   residual_out: torch.Tensor, normed: torch.Tensor | None = None,
                   post_gamma: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                   pre_gamma: torch.Tensor | None = None, inv_rms: torch.Tensor | None = None,
                   eps: float = 1e-6, residual_scale: float = 1.0,
                   ctx: Context | None = None) -> torch.Tensor:
    """The end of an expert block in one kernel (rr_unpermute_norm):

      c = sum_k route_weights[t, k] * y_permuted[route_pos[t, k]]
      residual_out = residual_scale * residual + gate * rms_norm(c) * post_gamma
      normed = rms_norm(residual_out) * pre_gamma

    y_permuted [T * top_k, N]; route_pos, route_weights [T, top_k]; residual,
    residual_out, normed [T, N] (residual_out may be residual); post_gamma,
    gate, pre_gamma float32 [N]. Without post_gamma c is not normalised, without
    gate it is not scaled, and normed goes with pre_gamma. inv_rms (float32
    [T, 2]) receives what the backward pass needs."""
    if ctx is None and (_calls or _load()).unpermute_norm(
            y_permuted, route_pos, route_weights, residual, post_gamma, gate, pre_gamma,
            residual_out, normed, inv_rms, eps, residual_scale):
        return residual_out
    dtype = _dtype(residual.dtype, "residual")
    sizes, inputs = _norm_inputs(y_permuted, route_pos, route_weights, residual, post_gamma, gate,
                                 pre_gamma)
    t, device, shape = residual.dtype, residual.device, residual.shape
    _call(lib().rr_unpermute_norm, "unpermute_norm", device, ctx, None, *inputs,
          _expect(residual_out, shape, t, device, "residual_out"),
          _expect(normed, shape, t, device, "normed"),
          _expect(inv_rms, (shape[0], 2), torch.float32, device, "inv_rms"), eps, residual_scale,
          *sizes, dtype)
    return residual_out


def unpermute_norm_backward_workspace_size(tokens: int, output: int) -> int:
    return int(lib().rr_unpermute_norm_backward_workspace_size(tokens, output))


def unpermute_norm_backward(y_permuted: torch.Tensor, route_pos: torch.Tensor,
                            route_weights: torch.Tensor, residual: torch.Tensor,
                            inv_rms: torch.Tensor | None, d_residual_out: torch.Tensor | None,
                            d_normed: torch.Tensor | None, d_residual: torch.Tensor,
                            d_y_permuted: torch.Tensor, d_route_weights: torch.Tensor,
                            post_gamma: torch.Tensor | None = None,
                            gate: torch.Tensor | None = None,
                            pre_gamma: torch.Tensor | None = None,
                            d_post_gamma: torch.Tensor | None = None,
                            d_gate: torch.Tensor | None = None,
                            d_pre_gamma: torch.Tensor | None = None,
                            residual_scale: float = 1.0,
                            workspace: torch.Tensor | None = None,
                            ctx: Context | None = None) -> None:
    """Gradients of unpermute_norm (rr_unpermute_norm_backward) from
    d_residual_out and d_normed (either may be None) and the saved inv_rms:
    d_residual [T, N] (may be d_residual_out), d_y_permuted [T * top_k, N],
    d_route_weights float32 [T, top_k] and the float32 [N] gradients of the
    parameters that are asked for."""
    if ctx is None and (_calls or _load()).unpermute_norm_backward(
            y_permuted, route_pos, route_weights, residual, post_gamma, gate, pre_gamma, inv_rms,
            d_residual_out, d_normed, d_residual, d_y_permuted, d_route_weights, d_post_gamma,
            d_gate, d_pre_gamma, residual_scale, workspace):
        return
    dtype = _dtype(residual.dtype, "residual")
    sizes, inputs = _norm_inputs(y_permuted, route_pos, route_weights, residual, post_gamma, gate,
                                 pre_gamma)
    tokens, top_k, output = sizes
    t, device, f32, shape = residual.dtype, residual.device, torch.float32, residual.shape
    _call(lib().rr_unpermute_norm_backward, "unpermute_norm_backward", device, ctx, workspace,
          *inputs, _expect(inv_rms, (tokens, 2), f32, device, "inv_rms"),
          _expect(d_residual_out, shape, t, device, "d_residual_out"),
          _expect(d_normed, shape, t, device, "d_normed"),
          _expect(d_residual, shape, t, device, "d_residual"),
          _expect(d_y_permuted, (tokens * top_k, output), t, device, "d_y_permuted"),
          _expect(d_route_weights, (tokens, top_k), f32, device, "d_route_weights"),
          _expect(d_post_gamma, (output,), f32, device, "d_post_gamma"),
          _expect(d_gate, (output,), f32, device, "d_gate"),
          _expect(d_pre_gamma, (output,), f32, device, "d_pre_gamma"), residual_scale, *sizes,
          dtype)
