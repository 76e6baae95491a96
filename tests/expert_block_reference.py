"""Plain float64 forms of the expert-block operators, and their inputs."""
from __future__ import annotations

import math

import numpy as np
import torch

ACTIVATIONS = ("silu", "gelu_tanh", "relu")


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def offsets_of(counts, device="cpu") -> torch.Tensor:
    return torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).to(device)


def random(shape, seed, device, dtype=torch.float32, std=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)


def act(name: str, g: torch.Tensor) -> torch.Tensor:
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return torch.clamp(g, min=0)


def gated(x, wg, wu, offsets, activation="silu"):
    """(g, u, h) in float64; rows outside every segment are zero."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    off = offsets.tolist()
    g = torch.zeros(x.shape[0], wg.shape[2], dtype=torch.float64, device=x.device)
    u = torch.zeros_like(g)
    for e, (a, b) in enumerate(zip(off, off[1:])):
        g[a:b] = x[a:b] @ wg[e]
        u[a:b] = x[a:b] @ wu[e]
    return g, u, act(activation, g) * u


def gated_backward(x, wg, wu, offsets, dh, activation="silu"):
    """(dx, dwg, dwu, dg, du) in float64."""
    x, wg, wu, dh = x.double(), wg.double(), wu.double(), dh.double()
    g, u, _ = gated(x, wg, wu, offsets)
    g = g.requires_grad_()
    a = act(activation, g)
    slope, = torch.autograd.grad(a.sum(), g)
    a = a.detach()
    dg, du = dh * u * slope, dh * a
    dx, dwg, dwu = torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)
    off = offsets.tolist()
    for e, (i, j) in enumerate(zip(off, off[1:])):
        dx[i:j] = dg[i:j] @ wg[e].T + du[i:j] @ wu[e].T
        dwg[e] = x[i:j].T @ dg[i:j]
        dwu[e] = x[i:j].T @ du[i:j]
    return dx, dwg, dwu, dg, du


def magnitudes(x, w, offsets):
    """sum_k |x||w| of every row and column: the scale of its rounding errors."""
    x, w = x.double().abs(), w.double().abs()
    off = offsets.tolist()
    out = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    for e, (a, b) in enumerate(zip(off, off[1:])):
        out[a:b] = x[a:b] @ w[e]
    return out


def unpermute_norm(yp, pos, weights, residual, post, gate, pre, eps, scale):
    """(residual_out, normed) in float64; invalid positions are skipped."""
    routes = yp.shape[0]
    pos = pos.long()
    there = (pos >= 0) & (pos < routes)
    rows = yp[pos.clamp(0, max(routes - 1, 0))] * there[..., None]
    c = (rows * (weights * there)[..., None]).sum(1)
    b = c if post is None else c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * post
    r = scale * residual + (b if gate is None else gate * b)
    n = None if pre is None else r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * pre
    return r, n


def normwise(got: torch.Tensor, want: torch.Tensor) -> float:
    want = want.double()
    got, want = got.detach().double(), want.detach()
    return float((got - want).norm() / want.norm().clamp(min=1e-300))
