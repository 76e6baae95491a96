"""The expert-block operators together, as a mixture-of-experts block uses them
beside the routing stages: router, gate, permute, gated projection, grouped
GEMM, combine with norms; in FP32 forward and backward, and in 8-bit integers.
"""
from __future__ import annotations

import math
import os
import subprocess
import sys

import torch
import pytest

import raggedroute_b200 as rr
from expert_block_reference import normwise, random, unpermute_norm

pytestmark = pytest.mark.gpu

T, K, E, N = 700, 192, 12, 160
EPS = 1e-6


def route(x, router):
    """Expert-grouped rows of x: (buffers, offsets, positions, weights)."""
    dev = x.device
    logits = torch.empty(T, E, device=dev)
    ids = torch.empty(T, 2, dtype=torch.int32, device=dev)
    w = torch.empty(T, 2, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    off = torch.empty(E + 1, dtype=torch.int32, device=dev)
    xp = torch.empty(2 * T, K, device=dev)
    pos = torch.empty(2 * T, dtype=torch.int32, device=dev)
    ws = torch.empty(rr.token_permute_workspace_size(T, E, 2, K), dtype=torch.uint8, device=dev)
    rr.dense_gemm(x, router, logits, T, E, K)
    rr.topk_gate(logits, ids, w, T, E)
    rr.histogram_exclusive_scan(ids, counts, off, 2 * T, E)
    rr.token_permute(x, ids, off, xp, pos, None, T, E, 2, K, ws)
    return ids, w, off, xp, pos.view(T, 2)


def make(device):
    return dict(x=random((T, K), 1, device), router=random((K, E), 2, device, std=K ** -0.5),
                wg=random((E, K, N), 3, device, std=K ** -0.5),
                wu=random((E, K, N), 4, device, std=K ** -0.5),
                wd=random((E, N, K), 5, device, std=N ** -0.5),
                post=random((K,), 6, device, std=0.1) + 1, gate=random((K,), 7, device, std=0.5),
                pre=random((K,), 8, device, std=0.1) + 1)


def test_fp32_block_forward_and_backward(cuda):
    m = make(cuda)
    ids, w, off, xp, pos = route(m["x"], m["router"])
    ws = torch.empty(rr.grouped_gated_gemm_workspace_size(2 * T, E, K, N, torch.float32, True),
                     dtype=torch.uint8, device=cuda)
    h, gu = torch.empty(2 * T, N, device=cuda), torch.empty(2 * T, 2 * N, device=cuda)
    yp = torch.empty(2 * T, K, device=cuda)
    out, normed = torch.empty(T, K, device=cuda), torch.empty(T, K, device=cuda)
    inv = torch.empty(T, 2, device=cuda)
    rr.grouped_gated_gemm(xp, m["wg"], m["wu"], off, h, gate_up=gu, workspace=ws)
    rr.grouped_gemm(h, m["wd"], off, yp, E, N, K, 2 * T)
    rr.unpermute_norm(yp, pos, w, m["x"], out, normed, post_gamma=m["post"], gate=m["gate"],
                      pre_gamma=m["pre"], inv_rms=inv, eps=EPS)

    # The same block token by token in float64, with the routing as decided.
    d = {k: v.double().requires_grad_() for k, v in m.items()}
    w64 = w.double().requires_grad_()
    rows = d["x"][torch.arange(T, device=cuda).repeat_interleave(2)]
    e = ids.view(-1).long()
    y = torch.zeros(2 * T, K, dtype=torch.float64, device=cuda)
    for i in range(E):
        at = (e == i).nonzero()[:, 0]
        g = rows[at] @ d["wg"][i]
        y = y.index_put((at,), (g * torch.sigmoid(g) * (rows[at] @ d["wu"][i])) @ d["wd"][i])
    order = torch.arange(2 * T, device=cuda).view(T, 2)
    want, want_n = unpermute_norm(y, order, w64, d["x"], d["post"], d["gate"], d["pre"], EPS, 1.0)
    # Three FP32 products in a row, each within 2^-19 normwise (grouped_gemm
    # within 1e-5), and a norm of bounded condition.
    assert normwise(out, want) < 3e-5 and normwise(normed, want_n) < 3e-5

    dro, dn = random((T, K), 9, cuda), random((T, K), 10, cuda)
    wsn = torch.empty(rr.unpermute_norm_backward_workspace_size(T, K), dtype=torch.uint8,
                      device=cuda)
    dres, dyp = torch.empty(T, K, device=cuda), torch.empty(2 * T, K, device=cuda)
    dw, dgate = torch.empty(T, 2, device=cuda), torch.empty(K, device=cuda)
    dpost, dpre = torch.empty(K, device=cuda), torch.empty(K, device=cuda)
    rr.unpermute_norm_backward(yp, pos, w, m["x"], inv, dro, dn, dres, dyp, dw,
                               post_gamma=m["post"], gate=m["gate"], pre_gamma=m["pre"],
                               d_post_gamma=dpost, d_gate=dgate, d_pre_gamma=dpre, workspace=wsn)
    # Through the down projection with the transposed weights, then the gated
    # projection; a token's rows of dx add up with weights of one.
    dh = torch.empty(2 * T, N, device=cuda)
    rr.grouped_gemm(dyp, m["wd"].transpose(1, 2).contiguous(), off, dh, E, K, N, 2 * T)
    dxp = torch.empty(2 * T, K, device=cuda)
    dwg, dwu = torch.empty_like(m["wg"]), torch.empty_like(m["wu"])
    rr.grouped_gated_gemm_backward(xp, m["wg"], m["wu"], off, gu, dh, dxp, dwg, dwu, workspace=ws)
    dx = torch.empty(T, K, device=cuda)
    rr.unpermute(dxp, pos.reshape(-1), torch.ones(2 * T, device=cuda), dx, T, 2, K)
    grads = torch.autograd.grad((want, want_n),
                                (d["x"], d["wg"], d["wu"], w64, d["post"], d["gate"], d["pre"]),
                                (dro.double(), dn.double()))
    got = (dx + dres, dwg, dwu, dw, dpost, dgate, dpre)
    for a, b in zip(got, grads):
        assert normwise(a, b) < 1e-4


def test_bf16_and_int8_block(cuda):
    """Rows grouped by the FP32 permute; the same block in bfloat16 with the
    permute on bfloat16 rows (viewed as half as many floats) and in integers."""
    m = make(cuda)
    ids, w, off, xp, pos = route(m["x"], m["router"])
    bf = torch.bfloat16
    xb = m["x"].to(bf)
    xpb = torch.empty(2 * T, K, dtype=bf, device=cuda)
    ws = torch.empty(rr.token_permute_workspace_size(T, E, 2, K // 2), dtype=torch.uint8,
                     device=cuda)
    flat = torch.empty(2 * T, dtype=torch.int32, device=cuda)
    rr.token_permute(xb.view(torch.float32), ids, off, xpb.view(torch.float32), flat, None, T, E,
                     2, K // 2, ws)
    assert torch.equal(xpb, xp.to(bf)) and torch.equal(flat.view(T, 2), pos)
    wg, wu = m["wg"].to(bf), m["wu"].to(bf)
    h = torch.empty(2 * T, N, dtype=bf, device=cuda)
    rr.grouped_gated_gemm(xpb, wg, wu, off, h)
    wq = torch.empty(E, K, rr.int8_row_stride(N), dtype=torch.int8, device=cuda)
    wsc = torch.empty(E, K, device=cuda)
    hq = torch.empty(2 * T, rr.int8_row_stride(N), dtype=torch.int8, device=cuda)
    hs = torch.empty(2 * T, device=cuda)
    yp = torch.empty(2 * T, K, dtype=bf, device=cuda)
    rr.quantize_expert_weights_int8(m["wd"], wq, wsc)
    rr.quantize_rows_int8(h, hq, hs)
    rr.grouped_gemm_int8(hq, hs, wq, wsc, off, yp)
    out, normed = torch.empty_like(xb), torch.empty_like(xb)
    rr.unpermute_norm(yp, pos, w, xb, out, normed, post_gamma=m["post"], gate=m["gate"],
                      pre_gamma=m["pre"], eps=EPS)
    o = off.tolist()
    y = torch.zeros(2 * T, K, dtype=torch.float64, device=cuda)
    for i, (a, b) in enumerate(zip(o, o[1:])):
        g = xpb[a:b].double() @ wg[i].double()
        y[a:b] = (g * torch.sigmoid(g) * (xpb[a:b].double() @ wu[i].double())) @ m["wd"][i].double()
    want, want_n = unpermute_norm(y, pos, w.double(), xb.double(), m["post"].double(),
                                  m["gate"].double(), m["pre"].double(), EPS, 1.0)
    # An 8-bit step is top / 127 with top below 6 deviations here: at most
    # 0.5 * 6 / 127 / sqrt(3) of a deviation per operand, two operands.
    assert normwise(out, want) < math.sqrt(2) * 3 / 127 / math.sqrt(3) + 2.0 ** -7
    assert normwise(normed, want_n) < math.sqrt(2) * 3 / 127 / math.sqrt(3) + 2.0 ** -7


def test_first_calls_inside_a_capture(cuda):
    """A process whose first calls are captured: nothing needs a plain call before."""
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "first_call_worker.py")
    run = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "first calls in a capture: ok" in run.stdout


def test_streams_side_by_side(cuda):
    """Calls on two streams at once, each with buffers and a workspace of its own."""
    results, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    bf = torch.bfloat16
    sets = []
    for i in range(2):
        x = random((3000, 264), 20 + i, cuda, bf)
        wg, wu = random((9, 264, 200), 30 + i, cuda, bf, 0.06), random((9, 264, 200), 40 + i, cuda,
                                                                     bf, 0.06)
        off = torch.tensor([0, 5, 5, 900, 1300, 1301, 1500, 2600, 2999, 3000],
                           dtype=torch.int32, device=cuda)
        size = rr.grouped_gated_gemm_workspace_size(3000, 9, 264, 200, bf, True)
        sets.append((x, wg, wu, off, random((3000, 200), 50 + i, cuda, bf),
                     torch.empty(size, dtype=torch.uint8, device=cuda)))

    def step(i):
        x, wg, wu, off, dh, ws = sets[i]
        h, gu = torch.empty_like(dh), torch.empty(3000, 400, device=cuda)
        dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
        rr.grouped_gated_gemm(x, wg, wu, off, h, gate_up=gu, workspace=ws)
        rr.grouped_gated_gemm_backward(x, wg, wu, off, gu, dh, dx, dwg, dwu, workspace=ws)
        return h, gu, dx, dwg, dwu

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results.append((i, step(i)))
    torch.cuda.synchronize()
    for i, got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def _calls(device, dtype):
    """Each operator as (function, its tensors by name, other arguments, outputs)."""
    t, k, n, e = 6, 32, 24, 3
    f32 = torch.float32

    def new(*shape, dtype=dtype):
        return torch.zeros(*shape, dtype=dtype, device=device)

    x, w = random((2 * t, k), 1, device, dtype=dtype), random((e, k, n), 2, device, dtype=dtype)
    off = torch.tensor([0, 5, 5, 2 * t], dtype=torch.int32, device=device)
    gated = dict(x_permuted=x, gate_weights=w, up_weights=w.clone(), offsets=off)
    gu = random((2 * t, 2 * n), 3, device)
    ws = new(rr.grouped_gated_gemm_workspace_size(2 * t, e, k, n, dtype, True), dtype=torch.uint8)
    yield (rr.grouped_gated_gemm, dict(gated, h=new(2 * t, n), gate_up=new(2 * t, 2 * n, dtype=f32),
                                       workspace=ws), dict(activation="gelu_tanh"), ["h", "gate_up"])
    yield (rr.grouped_gated_gemm_backward,
           dict(gated, gate_up=gu, dh=random((2 * t, n), 4, device, dtype=dtype), dx=new(2 * t, k),
                d_gate_weights=new(e, k, n), d_up_weights=new(e, k, n), workspace=ws),
           dict(activation="relu"), ["dx", "d_gate_weights", "d_up_weights"])
    xq, xs = new(2 * t, k, dtype=torch.int8), new(2 * t, dtype=f32)
    yield rr.quantize_rows_int8, dict(x=x, xq=xq, x_scale=xs), {}, ["xq", "x_scale"]
    wq, sc = new(e, n, k, dtype=torch.int8), new(e, n, dtype=f32)
    rr.quantize_expert_weights_int8(w, wq, sc)
    yield (rr.grouped_gemm_int8, dict(xq=xq, x_scale=xs, wq=wq, w_scale=sc, offsets=off,
                                      y_permuted=new(2 * t, n)), {}, ["y_permuted"])
    norm = dict(y_permuted=random((2 * t, n), 5, device, dtype=dtype),
                route_pos=torch.arange(2 * t, device=device).flip(0).int().view(t, 2),
                route_weights=random((t, 2), 6, device), residual=random((t, n), 7, device, dtype=dtype),
                post_gamma=random((n,), 8, device), gate=random((n,), 9, device),
                pre_gamma=random((n,), 10, device))
    inv = new(t, 2, dtype=f32)
    yield (rr.unpermute_norm, dict(norm, residual_out=new(t, n), normed=new(t, n), inv_rms=inv),
           dict(eps=1e-3, residual_scale=0.5), ["residual_out", "normed", "inv_rms"])
    grads = dict(d_residual=new(t, n), d_y_permuted=new(2 * t, n),
                 d_route_weights=new(t, 2, dtype=f32), d_post_gamma=new(n, dtype=f32),
                 d_gate=new(n, dtype=f32), d_pre_gamma=new(n, dtype=f32))
    yield (rr.unpermute_norm_backward,
           dict(norm, inv_rms=inv, d_residual_out=random((t, n), 11, device, dtype=dtype),
                d_normed=random((t, n), 12, device, dtype=dtype), **grads,
                workspace=new(rr.unpermute_norm_backward_workspace_size(t, n), dtype=torch.uint8)),
           dict(residual_scale=0.5), list(grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_compiled_and_plain_calls(cuda, dtype, monkeypatch):
    """A call through the compiled binding does what the Python one does, and
    what the binding declines is named by the Python one."""
    from raggedroute_b200 import expert_block

    def unused(*_):
        raise AssertionError("the Python path ran")

    plain_call = expert_block._call
    for fn, tensors, rest, outputs in _calls(cuda, dtype):
        with monkeypatch.context() as m:
            m.setattr(expert_block, "_call", unused)
            fn(**tensors, **rest)
        got = {k: tensors[k].clone() for k in outputs}
        assert all(v.any() for v in got.values()), fn.__name__
        for k in outputs:
            tensors[k].zero_()
        fn(**tensors, **rest, ctx=rr.Context())
        for k in outputs:
            assert torch.equal(got[k], tensors[k]), (fn.__name__, k)
        assert expert_block._call is plain_call
        for k, v in tensors.items():
            if k == "workspace":
                continue
            wrong = [torch.cat([v, v]), v.cpu(), v.double(),
                     torch.cat([v, v], -1).as_strided(v.shape, [2 * s for s in v.stride()])]
            for i, bad in enumerate(wrong):
                with pytest.raises((TypeError, ValueError)):
                    fn(**{**tensors, k: bad}, **rest)
        last = outputs[0]
        source = next(k for k, v in tensors.items() if k not in outputs and k != "workspace"
                      and v.dtype == tensors[last].dtype and v.numel() == tensors[last].numel()) \
            if fn is rr.unpermute_norm_backward else None
        if source is not None:  # an output that is an input: refused by the entry point
            with pytest.raises(rr.RaggedRouteError, match="unpermute_norm_backward: INVALID"):
                fn(**{**tensors, last: tensors[source]}, **rest)
    torch.cuda.synchronize()


def test_compiled_call_uses_the_current_stream(cuda):
    fn, tensors, rest, outputs = next(_calls(cuda, torch.float32))
    fn(**tensors, **rest)
    want = tensors["h"].clone()
    tensors["h"].zero_()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        fn(**tensors, **rest)
    assert not tensors["h"].any()  # captured, not run
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tensors["h"], want)


def test_captured_over_two_streams(cuda):
    """Kernels that start behind a fork, a copy, a memset and a join of streams,
    as captured and replayed with new inputs."""
    t, n = 700, 512
    yp, res = random((2 * t, n), 1, cuda), random((t, n), 2, cuda)
    pos = torch.randperm(2 * t, device=cuda).int().view(t, 2)
    w, ones = random((t, 2), 3, cuda), torch.ones(n, device=cuda)
    q, sc = torch.empty(t, n, dtype=torch.int8, device=cuda), torch.empty(t, device=cuda)
    bufs = [torch.empty(t, n, device=cuda) for _ in range(5)]
    q2, sc2 = torch.empty_like(q), torch.empty_like(sc)

    def run(side):
        main = torch.cuda.current_stream()
        a, an, b, bn, c = bufs
        rr.unpermute_norm(yp, pos, w, res, a, an, post_gamma=ones, pre_gamma=ones)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            rr.quantize_rows_int8(an, q, sc)           # behind the fork
            c.copy_(an)
            rr.unpermute_norm(yp, pos, w, c, c)        # behind a copy, in place
        rr.unpermute_norm(yp, pos, w, a, b, bn, gate=ones, pre_gamma=ones)
        main.wait_stream(side)
        rr.unpermute_norm(yp, pos, w, c, bn, residual_scale=0.5)  # behind the join
        c.zero_()
        rr.quantize_rows_int8(bn, q2, sc2)             # behind a memset

    side = torch.cuda.Stream()
    run(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(side)
    for seed in range(3):
        yp.copy_(random((2 * t, n), 10 + seed, cuda))
        res.copy_(random((t, n), 20 + seed, cuda))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*bufs, q, sc, q2, sc2)]
        run(side)
        torch.cuda.synchronize()
        assert all(torch.equal(g, x) for g, x in zip(got, (*bufs, q, sc, q2, sc2)))
        # The eager pass, kernel by kernel.
        a = torch.empty_like(res)
        an = torch.empty_like(res)
        rr.unpermute_norm(yp, pos, w, res, a, an, post_gamma=ones, pre_gamma=ones)
        torch.cuda.synchronize()
        c = an.clone()
        torch.cuda.synchronize()
        rr.unpermute_norm(yp, pos, w, c, c)
        torch.cuda.synchronize()
        last = torch.empty_like(c)
        rr.unpermute_norm(yp, pos, w, c, last, residual_scale=0.5)
        torch.cuda.synchronize()
        assert torch.equal(bufs[3], last) and torch.equal(bufs[0], a)


def test_chain_of_calls_with_no_pause(cuda):
    """Kernels of a long run of dependent calls start behind one another; each
    reads what the one before it wrote (and overwrites what it read)."""
    t, n = 3, 4096
    yp = random((2 * t, n), 1, cuda, std=0.1)
    pos = torch.arange(2 * t, device=cuda).int().view(t, 2)
    w, ones = random((t, 2), 2, cuda), torch.ones(n, device=cuda)
    start = random((t, n), 3, cuda)

    def run(pause):
        x = start.clone()
        q, sc = torch.empty(t, n, dtype=torch.int8, device=cuda), torch.empty(t, device=cuda)
        normed = torch.empty_like(x)
        out = []
        for i in range(200):
            rr.unpermute_norm(yp, pos, w, x, x, normed, post_gamma=ones, pre_gamma=ones)
            if pause:
                torch.cuda.synchronize()
            rr.quantize_rows_int8(normed, q, sc)
            if pause:
                torch.cuda.synchronize()
            rr.unpermute_norm(yp, pos, w, normed, x, residual_scale=0.9)
            if i % 50 == 49:
                out += [x.clone(), q.clone(), sc.clone()]
        return out

    want, got = run(True), run(False)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_graph_of_the_library(cuda, dtype):
    """Captured and replayed through raggedroute_b200.Graph."""
    for fn, tensors, rest, outputs in _calls(cuda, dtype):
        fn(**tensors, **rest)
        want = {k: tensors[k].clone() for k in outputs}
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        graph = rr.Graph.capture(lambda ctx: fn(**{k: v for k, v in tensors.items()}, **rest,
                                                ctx=ctx), stream)
        for k in outputs:
            tensors[k].zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.launch(stream)
        torch.cuda.synchronize()
        for k in outputs:
            assert torch.equal(tensors[k], want[k]), (fn.__name__, k)
