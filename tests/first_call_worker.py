"""Makes the expert-block operators' first calls of a process inside a stream
capture, replays them and compares with plain calls. Run by
test_gpu_expert_block.py in a process of its own."""
from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import raggedroute_b200 as rr  # noqa: E402

dev, bf = torch.device("cuda:0"), torch.bfloat16
R, E, K, N, T = 800, 5, 128, 96, 700
torch.manual_seed(0)
x = torch.randn(R, K, device=dev, dtype=bf)
wg, wu = torch.randn(E, K, N, device=dev, dtype=bf), torch.randn(E, K, N, device=dev, dtype=bf)
off = torch.tensor([0, 300, 300, 301, 620, 800], dtype=torch.int32, device=dev)
h, gu = torch.zeros(R, N, device=dev, dtype=bf), torch.zeros(R, 2 * N, device=dev)
dh, dx = torch.randn(R, N, device=dev, dtype=bf), torch.zeros_like(x)
dwg, dwu = torch.zeros_like(wg), torch.zeros_like(wu)
wq, ws = torch.zeros(E, N, K, dtype=torch.int8, device=dev), torch.zeros(E, N, device=dev)
xq, xs = torch.zeros(R, K, dtype=torch.int8, device=dev), torch.zeros(R, device=dev)
y = torch.zeros(R, N, device=dev, dtype=bf)
yp, res = torch.randn(2 * T, 4096, device=dev, dtype=bf), torch.randn(T, 4096, device=dev, dtype=bf)
pos = torch.randperm(2 * T, device=dev).to(torch.int32).view(T, 2)
w = torch.rand(T, 2, device=dev)
gamma = torch.rand(3, 4096, device=dev)
out, normed, inv = torch.zeros_like(res), torch.zeros_like(res), torch.zeros(T, 2, device=dev)
dres, dyp, dw = torch.zeros_like(res), torch.zeros_like(yp), torch.zeros(T, 2, device=dev)
dgamma = torch.zeros(3, 4096, device=dev)
buf = torch.zeros(1 << 24, dtype=torch.uint8, device=dev)
results = (h, gu, dx, dwg, dwu, wq, ws, xq, xs, y, out, normed, inv, dres, dyp, dw, dgamma)


def step(ctx):
    rr.grouped_gated_gemm(x, wg, wu, off, h, gate_up=gu, workspace=buf, ctx=ctx)
    rr.grouped_gated_gemm_backward(x, wg, wu, off, gu, dh, dx, dwg, dwu, workspace=buf, ctx=ctx)
    rr.quantize_expert_weights_int8(wg, wq, ws, ctx=ctx)
    rr.quantize_rows_int8(x, xq, xs, ctx=ctx)
    rr.grouped_gemm_int8(xq, xs, wq, ws, off, y, ctx=ctx)
    rr.unpermute_norm(yp, pos, w, res, out, normed, post_gamma=gamma[0], gate=gamma[1],
                      pre_gamma=gamma[2], inv_rms=inv, ctx=ctx)
    rr.unpermute_norm_backward(yp, pos, w, res, inv, res, normed, dres, dyp, dw,
                               post_gamma=gamma[0], gate=gamma[1], pre_gamma=gamma[2],
                               d_post_gamma=dgamma[0], d_gate=dgamma[1], d_pre_gamma=dgamma[2],
                               workspace=buf, ctx=ctx)


stream = torch.cuda.Stream()
torch.cuda.synchronize()
graph = rr.Graph.capture(step, stream)
graph.launch(stream)
stream.synchronize()
captured = [t.clone() for t in results]
step(None)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, results))
assert all(t.float().abs().sum() > 0 for t in results)
print("first calls in a capture: ok")
