"""Workloads of the expert-block operators: the gated expert projection and its
backward pass, the 8-bit integer grouped product, and the weighted combine with
the norms, gate and residual around an expert block and its backward pass.

A case is a dict of sizes. `prepare` makes its inputs on the GPU, `run` makes one
pass (in elementary torch operations, or through raggedroute_b200 when `own` is
set), `exact` evaluates the operator's definition in float64, and `work` counts
the bytes and operations a pass cannot do without.

Definitions. Rows are grouped by expert: segment e is rows [offsets[e],
offsets[e+1]).
  gated        g = x Wg[e], u = x Wu[e], h = act(g) * u
  gated_train  the same, then from dh: dg = dh*u*act'(g), du = dh*act(g),
               dx = dg Wg[e]^T + du Wu[e]^T, dWg[e] = x^T dg, dWu[e] = x^T du
  int8         per row: s = max|x| / 127, q = rint(x * (127 / max|x|)); then
               y = (q . wq[e]^T) * s * ws[e], wq and ws given
  norm         c = sum_k w_k yp[pos_k], b = c * rsqrt(mean(c^2) + eps) * post,
               r' = scale * r + gate * b, n = r' * rsqrt(mean(r'^2) + eps) * pre
  norm_train   the same, then every gradient from (dr', dn)
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One decoded token of the 128-expert layer: two routes, bound by the
        # weights of two experts and by latency.
        dict(name="gated_one_token", op="gated", dtype="bf16", tokens=1, top_k=2, experts=128,
             hidden=4096, output=1408, empty=0),
        # The prefill of that layer: the largest product.
        dict(name="gated_prefill", op="gated", dtype="bf16", tokens=65536, top_k=2, experts=128,
             hidden=4096, output=1408, empty=0),
        # The same operator at the strict FP32 contract of the grouped GEMM
        # (32768 routes over 64 experts, some of them empty).
        dict(name="gated_fp32", op="gated", dtype="fp32", tokens=16384, top_k=2, experts=64,
             hidden=1024, output=1024, empty=6),
        # A training step of one expert-parallel rank's share of the layer.
        dict(name="gated_train", op="gated_train", dtype="bf16", tokens=16384, top_k=2, experts=16,
             hidden=4096, output=1408, empty=0),
        # A small FP32 training step (the 4096-token chain's sizes).
        dict(name="gated_train_fp32", op="gated_train", dtype="fp32", tokens=4096, top_k=2,
             experts=64, hidden=256, output=128, empty=3),
        # Sizes that are no multiple of any tile, vector or alignment.
        dict(name="gated_train_odd", op="gated_train", dtype="bf16", tokens=5003, top_k=1,
             experts=17, hidden=1001, output=333, empty=2),
        # 8-bit serving: one token, a prefill, and ragged odd sizes from FP32 rows.
        dict(name="int8_one_token", op="int8", dtype="bf16", tokens=1, top_k=2, experts=128,
             hidden=4096, output=1408, empty=0),
        dict(name="int8_prefill", op="int8", dtype="bf16", tokens=65536, top_k=2, experts=128,
             hidden=4096, output=1408, empty=0),
        dict(name="int8_odd", op="int8", dtype="fp32", tokens=2051, top_k=2, experts=33,
             hidden=1030, output=515, empty=1),
        # The end of an expert block for one token, and for a training batch.
        dict(name="norm_one_token", op="norm", dtype="bf16", tokens=1, top_k=2, output=4096),
        dict(name="norm_fp32", op="norm", dtype="fp32", tokens=16384, top_k=2, output=1024),
        dict(name="norm_train", op="norm_train", dtype="bf16", tokens=32768, top_k=2,
             output=4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gated", "gated_train", "int8", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op.startswith("norm"):
        n = _log(rng, 64, 8192)
        t = min(_log(rng, 1, 65536), 32768 * 4096 // n)
        return dict(op=op, dtype=dtype, tokens=max(1, t), top_k=rng.choice([2, 2, 4, 8]),
                    output=n) if t * n <= 1 << 25 else \
            dict(op=op, dtype=dtype, tokens=t, top_k=2, output=n)
    e = _log(rng, 1, 128)
    k = _log(rng, 64, 4096)
    n = _log(rng, 32, 1408)
    if rng.random() < 0.6:  # sizes of real layers: multiples of 64
        k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
    top_k = rng.choice([1, 2, 2])
    most = 32768 if op == "gated_train" else 131072
    if dtype == "fp32":
        most //= 4
    t = max(1, min(_log(rng, 1, 65536), most // top_k))
    return dict(op=op, dtype=dtype, tokens=t, top_k=top_k, experts=e, hidden=k, output=n,
                empty=rng.choice([0, 0, 1]) if e > 2 else 0)


def _counts(case, seed):
    """Rows of each expert: a balanced router's spread, `empty` experts idle."""
    r = np.random.default_rng(seed)
    e = case["experts"]
    p = np.exp(0.2 * r.standard_normal(e))
    p[r.permutation(e)[: case["empty"]]] = 0.0
    return r.multinomial(case["tokens"] * case["top_k"], p / p.sum())


def prepare(case, seed):
    dt, dev = TYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype).mul_(std)

    t, n = case["tokens"], case["output"]
    r = t * case["top_k"]
    s = dict(case=case)
    if case["op"].startswith("norm"):
        order = torch.randperm(r, generator=g, device=dev)
        s["route_pos"] = order.to(torch.int32).view(t, -1)
        s["route_weights"] = torch.softmax(normal(t, case["top_k"], dtype=torch.float32), 1)
        s["yp"] = normal(r, n, std=0.5)
        s["residual"] = normal(t, n)
        s["post"] = normal(n, std=0.1, dtype=torch.float32).add_(1.0)
        s["pre"] = normal(n, std=0.1, dtype=torch.float32).add_(1.0)
        s["gate"] = normal(n, std=0.3, dtype=torch.float32)
        s["scale"] = 1.0
        s["residual_out"], s["normed"] = torch.empty(t, n, device=dev, dtype=dt), \
            torch.empty(t, n, device=dev, dtype=dt)
        if case["op"] == "norm_train":
            s["d_residual_out"] = normal(t, n)
            s["d_normed"] = normal(t, n)
            s["inv_rms"] = torch.empty(t, 2, device=dev, dtype=torch.float32)
            s["d_residual"] = torch.empty(t, n, device=dev, dtype=dt)
            s["d_yp"] = torch.empty(r, n, device=dev, dtype=dt)
            s["d_weights"] = torch.empty(t, case["top_k"], device=dev, dtype=torch.float32)
            for name in ("d_post", "d_gate", "d_pre"):
                s[name] = torch.empty(n, device=dev, dtype=torch.float32)
        return s
    e, k = case["experts"], case["hidden"]
    counts = _counts(case, seed)
    s["max_rows"] = int(counts.max())
    s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).to(dev)
    s["x"] = normal(r, k)
    if case["op"] == "int8":
        # Weights quantised ahead: [experts, output, hidden rounded up to 16],
        # zero-filled, one scale for each output channel.
        wide = (k + 15) // 16 * 16
        s["wq"] = torch.zeros(e, n, wide, device=dev, dtype=torch.int8)
        s["wq"][:, :, :k] = torch.randint(-127, 128, (e, n, k), generator=g, device=dev,
                                          dtype=torch.int8)
        s["ws"] = torch.rand(e, n, generator=g, device=dev).add_(0.5).mul_(
            3.0 / (127 * math.sqrt(k)))
        s["xq"] = torch.empty(r, wide, device=dev, dtype=torch.int8)
        s["xs"] = torch.empty(r, device=dev, dtype=torch.float32)
        s["y"] = torch.empty(r, n, device=dev, dtype=dt)
        return s
    s["wg"] = normal(e, k, n, std=1.0 / math.sqrt(k))
    s["wu"] = normal(e, k, n, std=1.0 / math.sqrt(k))
    s["h"] = torch.empty(r, n, device=dev, dtype=dt)
    if case["op"] == "gated_train":
        s["dh"] = normal(r, n, std=1.0 / math.sqrt(n))
        s["gate_up"] = torch.empty(r, 2 * n, device=dev, dtype=torch.float32)
        s["dx"] = torch.empty(r, k, device=dev, dtype=dt)
        s["dwg"], s["dwu"] = torch.empty(e, k, n, device=dev, dtype=dt), \
            torch.empty(e, k, n, device=dev, dtype=dt)
    return s


# ---- plain forms ------------------------------------------------------------

def _groups(s):
    """Row of each (expert, slot), whether it is there, and each row's place."""
    off = s["offsets"].long()
    r = s["x"].shape[0]
    at = off[:-1, None] + torch.arange(s["max_rows"], device=off.device)
    rows = torch.arange(r, device=off.device)
    expert = torch.searchsorted(off[1:], rows, right=True)
    return at.clamp(max=r - 1), at < off[1:, None], expert, rows - off[expert]


def _few(s):
    """Fewer rows than experts: a row takes its own expert's weights."""
    return s["x"].shape[0] <= s["offsets"].numel() - 1


def _grouped(a, w, groups):
    """a[r] . w[expert of r] for every row, over padded groups."""
    at, there, expert, slot = groups
    return torch.bmm(a[at] * there[..., None], w)[expert, slot]


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain_gated(s):
    x = s["x"].float()
    groups = _groups(s)
    if _few(s):
        e = groups[2]
        g = torch.bmm(x[:, None], s["wg"][e].float())[:, 0]
        u = torch.bmm(x[:, None], s["wu"][e].float())[:, 0]
    else:
        g = _grouped(x, s["wg"].float(), groups)
        u = _grouped(x, s["wu"].float(), groups)
    return g, u, (_silu(g) * u).to(s["x"].dtype)


def _plain_gated_train(s):
    g, u, h = _plain_gated(s)
    dt = s["x"].dtype
    at, there, _, _ = groups = _groups(s)
    dh = s["dh"].float()
    sig = 1.0 / (1.0 + torch.exp(-g))
    dg = dh * u * sig * (1.0 + g * (1.0 - sig))
    du = dh * g * sig
    dx = _grouped(dg, s["wg"].float().mT, groups) + _grouped(du, s["wu"].float().mT, groups)
    xt = (s["x"].float()[at] * there[..., None]).mT
    dwg = torch.bmm(xt, dg[at] * there[..., None])
    dwu = torch.bmm(xt, du[at] * there[..., None])
    return dict(h=h, dx=dx.to(dt), dwg=dwg.to(dt), dwu=dwu.to(dt))


def _quantized(x):
    """Scaled rows in whole numbers, and each row's scale, in 32 bits."""
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(x * (torch.full_like(top, 127.0) / top))
    return q, top / torch.full_like(top, 127.0)


def _plain_int8(s):
    q, scale = _quantized(s["x"].float())
    k = q.shape[1]
    groups = _groups(s)
    e = groups[2]
    if _few(s):
        y = torch.bmm(q[:, None], s["wq"][e][:, :, :k].float().mT)[:, 0]
    else:
        y = _grouped(q, s["wq"][:, :, :k].float().mT, groups)
    return dict(y=(y * scale * s["ws"][e]).to(s["x"].dtype), scale=scale[:, 0])


def _plain_norm(s):
    dt = s["yp"].dtype
    rows = s["yp"].float()[s["route_pos"].long()]
    c = (rows * s["route_weights"][..., None]).sum(1)
    i1 = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    b = c * i1 * s["post"]
    r = s["scale"] * s["residual"].float() + s["gate"] * b
    i2 = torch.rsqrt((r * r).mean(1, keepdim=True) + EPS)
    return rows, c, i1, b, r, i2, dict(residual_out=r.to(dt), normed=(r * i2 * s["pre"]).to(dt))


def _plain_norm_train(s):
    dt = s["yp"].dtype
    rows, c, i1, b, r, i2, out = _plain_norm(s)
    dn = s["d_normed"].float()
    v = dn * s["pre"]
    rn = r * i2
    dr = s["d_residual_out"].float() + i2 * (v - rn * (v * rn).mean(1, keepdim=True))
    db = dr * s["gate"]
    cn = c * i1
    v = db * s["post"]
    dc = i1 * (v - cn * (v * cn).mean(1, keepdim=True))
    d_yp = torch.empty_like(s["yp"])
    d_yp[s["route_pos"].long()] = (dc[:, None] * s["route_weights"][..., None]).to(dt)
    out.update(d_residual=(s["scale"] * dr).to(dt), d_yp=d_yp,
               d_weights=(rows * dc[:, None]).sum(2),
               d_post=(db * cn).double().sum(0).float(), d_gate=(dr * b).double().sum(0).float(),
               d_pre=(dn * rn).double().sum(0).float())
    return out


# ---- the framework's calls ---------------------------------------------------

def _workspace(s, size):
    """A program's workspace, kept as long as its buffers."""
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(size, 256), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _own(s):
    import raggedroute_b200 as rr
    op = s["case"]["op"]
    if op == "gated":
        x, w = s["x"], s["wg"]
        ws = _workspace(s, rr.grouped_gated_gemm_workspace_size(
            x.shape[0], w.shape[0], w.shape[1], w.shape[2], x.dtype))
        rr.grouped_gated_gemm(x, w, s["wu"], s["offsets"], s["h"], activation="silu",
                              workspace=ws)
        return dict(h=s["h"])
    if op == "gated_train":
        x, w = s["x"], s["wg"]
        ws = _workspace(s, rr.grouped_gated_gemm_workspace_size(
            x.shape[0], w.shape[0], w.shape[1], w.shape[2], x.dtype, backward=True))
        rr.grouped_gated_gemm(x, w, s["wu"], s["offsets"], s["h"], gate_up=s["gate_up"],
                              activation="silu", workspace=ws)
        rr.grouped_gated_gemm_backward(x, w, s["wu"], s["offsets"], s["gate_up"], s["dh"],
                                       s["dx"], s["dwg"], s["dwu"], activation="silu",
                                       workspace=ws)
        return dict(h=s["h"], dx=s["dx"], dwg=s["dwg"], dwu=s["dwu"])
    if op == "int8":
        rr.quantize_rows_int8(s["x"], s["xq"], s["xs"])
        rr.grouped_gemm_int8(s["xq"], s["xs"], s["wq"], s["ws"], s["offsets"], s["y"])
        return dict(y=s["y"], scale=s["xs"])
    train = op == "norm_train"
    rr.unpermute_norm(s["yp"], s["route_pos"], s["route_weights"], s["residual"],
                      s["residual_out"], s["normed"], post_gamma=s["post"], gate=s["gate"],
                      pre_gamma=s["pre"], inv_rms=s["inv_rms"] if train else None, eps=EPS,
                      residual_scale=s["scale"])
    out = dict(residual_out=s["residual_out"], normed=s["normed"])
    if train:
        ws = _workspace(s, rr.unpermute_norm_backward_workspace_size(*s["residual"].shape))
        rr.unpermute_norm_backward(s["yp"], s["route_pos"], s["route_weights"], s["residual"],
                                   s["inv_rms"], s["d_residual_out"], s["d_normed"],
                                   s["d_residual"], s["d_yp"], s["d_weights"],
                                   post_gamma=s["post"], gate=s["gate"], pre_gamma=s["pre"],
                                   d_post_gamma=s["d_post"], d_gate=s["d_gate"],
                                   d_pre_gamma=s["d_pre"], residual_scale=s["scale"],
                                   workspace=ws)
        out.update({k: s[k] for k in ("d_residual", "d_yp", "d_weights", "d_post", "d_gate",
                                      "d_pre")})
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "gated":
        return dict(h=_plain_gated(state)[2])
    if op == "gated_train":
        return _plain_gated_train(state)
    if op == "int8":
        return _plain_int8(state)
    if op == "norm":
        return _plain_norm(state)[-1]
    return _plain_norm_train(state)


# ---- the definition in 64 bits -----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(case, s)
    off = s["offsets"].tolist()
    r, k, n = s["x"].shape[0], case["hidden"], case["output"]

    def new(*shape):
        return torch.zeros(*shape, device="cuda", dtype=torch.float64)

    if case["op"] == "int8":
        y = new(r, n)
        x32 = s["x"].float()
        top = x32.abs().max(dim=1).values
        # The scaled value is rounded in 32 bits by definition.
        q = (x32 * (torch.full_like(top, 127.0) / top)[:, None]).round().double()
        scale = top.double() / 127.0
        for e, (a, b) in enumerate(zip(off, off[1:])):
            if b > a:
                y[a:b] = (q[a:b] @ s["wq"][e, :, :k].double().T) * scale[a:b, None] \
                    * s["ws"][e].double()
        return dict(y=y, scale=scale)
    train = case["op"] == "gated_train"
    out = dict(h=new(r, n))
    if train:
        out.update(dx=new(r, k), dwg=new(case["experts"], k, n), dwu=new(case["experts"], k, n))
    for e, (a, b) in enumerate(zip(off, off[1:])):
        if b == a:
            continue
        x, wg, wu = s["x"][a:b].double(), s["wg"][e].double(), s["wu"][e].double()
        g, u = x @ wg, x @ wu
        sig = torch.sigmoid(g)
        out["h"][a:b] = g * sig * u
        if train:
            dh = s["dh"][a:b].double()
            dg, du = dh * u * (sig + g * sig * (1 - sig)), dh * g * sig
            out["dx"][a:b] = dg @ wg.T + du @ wu.T
            out["dwg"][e], out["dwu"][e] = x.T @ dg, x.T @ du
    return out


def _exact_norm(case, s):
    t, n = case["tokens"], case["output"]
    yp = s["yp"].double().requires_grad_()
    w = s["route_weights"].double().requires_grad_()
    res = s["residual"].double().requires_grad_()
    post, gate, pre = (s[v].double().requires_grad_() for v in ("post", "gate", "pre"))
    c = torch.zeros(t, n, device="cuda", dtype=torch.float64)
    for j in range(case["top_k"]):
        c = c + w[:, j, None] * yp[s["route_pos"][:, j].long()]
    b = post * c / torch.sqrt(c.pow(2).sum(1, keepdim=True) / n + EPS)
    ro = s["scale"] * res + gate * b
    normed = pre * ro / torch.sqrt(ro.pow(2).sum(1, keepdim=True) / n + EPS)
    out = dict(residual_out=ro.detach(), normed=normed.detach())
    if case["op"] == "norm_train":
        grads = torch.autograd.grad((ro, normed), (res, yp, w, post, gate, pre),
                                    (s["d_residual_out"].double(), s["d_normed"].double()))
        out.update(zip(("d_residual", "d_yp", "d_weights", "d_post", "d_gate", "d_pre"), grads))
    return out


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    t, n = case["tokens"], case["output"]
    r = t * case["top_k"]
    if case["op"].startswith("norm"):
        train = case["op"] == "norm_train"
        # forward: rows, residual in; residual_out, normed out. backward: rows
        # and residual are read once for both passes; two gradients in, two out.
        moved = (r + 3 * t) * n * size + 8 * r + 12 * n
        if train:
            moved += (r + 3 * t) * n * size + 4 * r + 12 * n
        return dict(bytes=moved, flops=(4 * r + (30 if train else 10) * t) * n)
    k = case["hidden"]
    active = min(case["experts"] - case["empty"], r)
    if case["op"] == "int8":
        return dict(bytes=r * k * size + active * n * (k + 4) + r * n * size + 4 * r,
                    flops=2 * r * k * n)
    moved = r * k * size + 2 * active * k * n * size + r * n * size
    if case["op"] == "gated":
        return dict(bytes=moved, flops=4 * r * k * n)
    moved += r * n * size + r * k * size + 2 * case["experts"] * k * n * size
    return dict(bytes=moved, flops=12 * r * k * n)
