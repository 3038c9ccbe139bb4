"""The 16-bit operators of a mixture-of-experts layer, as cases to measure.

An NVFP4 model keeps some of its layers in bf16 or fp16 (the first and last blocks, the
output projections, the experts while they are trained or calibrated), and around the
experts' products it needs the router and the movement of token rows to their experts and
back.  Four operators cover that:

  linear   Y = act(X W^T + bias) + residual, and its gradients
  grouped  the same product by expert over ragged row groups, and its gradients
  route    top-k expert choice: weights, experts, row of each (token, choice), row offsets;
           and the gradient of the logits
  move     token rows gathered into expert order (dispatch) and summed back with the
           routing weights (combine), and the gradients of both

Each case runs in a plain form (elementary torch operations in 32 bits, rounded once at the
end) or, where `own` is true, through the nvfp4_b200 package.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LARGEST_FLOPS = 2.0 * 8192 * 28672 * 4096  # the largest listed case


def _nv():
    import os
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-kernels_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nvfp4_b200
    return nvfp4_b200


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through an attention output projection with bias and residual: the
        # latency of a decode step
        dict(name="linear decode M1", op="linear", train=False, M=1, N=4096, K=4096, act="none", bias=True,
             residual=True, dtype="bf16"),
        # a short ragged prompt through an MLP's first layer, sizes that fill no tile
        dict(name="linear ragged M333", op="linear", train=False, M=333, N=14344, K=4104, act="gelu_tanh",
             bias=True, residual=False, dtype="fp16"),
        # a long prompt through a square projection added to the residual stream
        dict(name="linear prefill 8192", op="linear", train=False, M=8192, N=8192, K=8192, act="none", bias=True,
             residual=True, dtype="bf16"),
        # training step of an MLP's first layer: gradients of input, weight and bias
        dict(name="linear train", op="linear", train=True, M=4096, N=14336, K=4096, act="gelu_tanh", bias=True,
             residual=False, dtype="bf16"),
        # 32 tokens x top-2 through 8 experts' gate and up projections: decoding in a batch
        dict(name="experts decode 64 rows", op="grouped", train=False, rows=64, G=8, N=28672, K=4096, act="swiglu",
             bias=False, empty=0, dtype="bf16"),
        # 4096 tokens x top-2 through the same experts: prefill
        dict(name="experts prefill 8192 rows", op="grouped", train=False, rows=8192, G=8, N=28672, K=4096,
             act="swiglu", bias=False, empty=0, dtype="bf16"),
        # training step of 64 small experts, some of them without a row
        dict(name="experts train 64", op="grouped", train=True, rows=16387, G=64, N=2048, K=2048, act="swiglu",
             bias=True, empty=5, dtype="bf16"),
        # the router of one decode step of a small batch
        dict(name="route decode", op="route", train=False, T=16, E=64, k=4, scoring="softmax", select_bias=False,
             renormalize=True, masked=0.0, dtype="bf16"),
        # the router of a long prefill with many experts, a balancing bias and padding tokens
        dict(name="route prefill", op="route", train=False, T=16381, E=256, k=8, scoring="sigmoid",
             select_bias=True, renormalize=True, masked=0.05, dtype="fp32"),
        # the router of a training step: choice and gradient of the logits
        dict(name="route train", op="route", train=True, T=4096, E=8, k=2, scoring="softmax", select_bias=False,
             renormalize=False, masked=0.0, dtype="bf16"),
        # rows of a decode step to their experts and back, with the residual
        dict(name="move decode", op="move", train=False, T=32, E=8, k=2, K=4096, residual=True, masked=0.0,
             dtype="bf16"),
        # rows of a training step to many experts and back, with the gradients
        dict(name="move train", op="move", train=True, T=8191, E=128, k=8, K=2048, residual=False, masked=0.02,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["linear", "grouped", "route", "move"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if op == "linear":
            act = rng.choice(["none", "relu", "silu", "gelu_tanh", "swiglu"])
            case = dict(op=op, train=rng.random() < 0.35, M=_log_int(rng, 1, 16384),
                        N=_log_int(rng, 256, 28672, 32 if act == "swiglu" else 8), K=_log_int(rng, 256, 16384, 8),
                        act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5, dtype=dtype)
            cost = work(case)["flops"]
        elif op == "grouped":
            act = rng.choice(["none", "relu", "silu", "swiglu", "swiglu"])
            G = _log_int(rng, 2, 128)
            case = dict(op=op, train=rng.random() < 0.35, rows=_log_int(rng, 2, 32768), G=G,
                        N=_log_int(rng, 256, 28672, 32 if act == "swiglu" else 8), K=_log_int(rng, 256, 8192, 8),
                        act=act, bias=rng.random() < 0.5, empty=rng.randrange(0, max(1, G // 4)), dtype=dtype)
            # the weights and their 32-bit copies have to fit beside the inputs of other passes
            if case["G"] * case["N"] * case["K"] > 8 * 28672 * 4096:
                continue
            cost = work(case)["flops"]
        elif op == "route":
            E = rng.choice([8, 16, 60, 64, 128, 160, 256])
            scoring = rng.choice(["softmax", "sigmoid"])
            case = dict(op=op, train=rng.random() < 0.35, T=_log_int(rng, 1, 32768), E=E,
                        k=rng.randint(1, min(8, E)), scoring=scoring,
                        select_bias=scoring == "sigmoid" and rng.random() < 0.5, renormalize=rng.random() < 0.6,
                        masked=rng.choice([0.0, 0.05]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
            cost = 0.0
        else:
            E = rng.choice([8, 16, 64, 128, 256])
            case = dict(op=op, train=rng.random() < 0.35, T=_log_int(rng, 1, 16384), E=E,
                        k=rng.randint(1, min(8, E)), K=_log_int(rng, 256, 8192, 8), residual=rng.random() < 0.5,
                        masked=rng.choice([0.0, 0.02]), dtype=dtype)
            if case["T"] * case["k"] * case["K"] > 8191 * 8 * 2048 * 2:
                continue
            cost = 0.0
        if cost <= _LARGEST_FLOPS:
            return case


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _weight(g, rows, K, dtype):
    w = torch.empty(rows, K, device="cuda", dtype=dtype)
    step = max(1, (1 << 27) // K)
    for r in range(0, rows, step):
        part = w[r:r + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(K ** -0.5))
    return w


def _group_sizes(case, seed):
    """Rows of each expert: an uneven routing (the fullest expert takes about 1.5 times the
    mean), `empty` of the experts without a row."""
    r = random.Random(seed * 7919 + case["rows"])
    G, rows = case["G"], case["rows"]
    none = set(r.sample(range(G), case["empty"]))
    share = [0.0 if g in none else r.uniform(0.5, 1.5) for g in range(G)]
    total, acc, cuts = sum(share), 0.0, [0]
    for s in share:
        acc += s
        cuts.append(int(round(rows * acc / total)))
    cuts[-1] = rows
    return cuts


def _logits(case, g):
    T, E = case["T"], case["E"]
    x = torch.randn(T, E, device="cuda", generator=g) * 2
    if case["masked"]:
        x.masked_fill_(torch.rand(T, E, device="cuda", generator=g) < case["masked"], -math.inf)
        x.masked_fill_(torch.rand(T, 1, device="cuda", generator=g) < case["masked"], -math.inf)  # padding tokens
    return x.to(_DT[case["dtype"]])


def prepare(case, seed):
    g = _gen(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    s = dict(case=case)
    if op in ("linear", "grouped"):
        M = case["M"] if op == "linear" else case["rows"]
        G = 1 if op == "linear" else case["G"]
        N, K = case["N"], case["K"]
        No = N // 2 if case["act"] == "swiglu" else N
        s["x"] = _normal(g, (M, K), dt)
        s["w"] = _weight(g, G * N, K, dt)
        if op == "grouped":
            cuts = _group_sizes(case, seed)
            s["m_offsets"] = torch.tensor(cuts, dtype=torch.int32, device="cuda")
            s["capacity"] = max(1, max(b - a for a, b in zip(cuts, cuts[1:])))
            s["cuts"] = cuts
        if case["train"]:
            s["dy"] = _normal(g, (M, No), dt)
            s["z"] = _normal(g, (M, N), dt) if case["act"] != "none" else None
        else:
            shape = (N,) if op == "linear" else (G, N)
            s["bias"] = _normal(g, shape, dt, 0.5) if case["bias"] else None
            s["residual"] = _normal(g, (M, No), dt) if case.get("residual") else None
    elif op == "route":
        s["logits"] = _logits(case, g)
        s["bias"] = torch.randn(case["E"], device="cuda", generator=g) * 0.05 if case["select_bias"] else None
        if case["train"]:
            s["dweights"] = torch.randn(case["T"], case["k"], device="cuda", generator=g)
    else:
        logits = _logits(dict(case, dtype="fp32"), g)
        s["routing"] = _plain_route(logits, case["k"], "softmax", None, True, 1.0)
        T, k, K = case["T"], case["k"], case["K"]
        s["x"] = _normal(g, (T, K), dt)
        s["expert_rows"] = _normal(g, (T * k, K), dt)
        s["residual"] = _normal(g, (T, K), dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = _normal(g, (T, K), dt)
            s["drows"] = _normal(g, (T * k, K), dt)
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if act == "swiglu":  # blocks of 16 gate columns, then 16 up columns
        v = z.unflatten(-1, (-1, 2, 16))
        gate, up = v[..., 0, :], v[..., 1, :]
        return (gate / (1 + torch.exp(-gate)) * up).flatten(-2)
    return z


def _plain_dact(dy, z, act):
    if act == "relu":
        return torch.where(z > 0, dy, torch.zeros_like(dy))
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return dy * (sg + z * sg * (1 - sg))
    if act == "gelu_tanh":
        c = 0.7978845608028654
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return dy * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z))
    if act == "swiglu":
        v, d = z.unflatten(-1, (-1, 2, 16)), dy.unflatten(-1, (-1, 16))
        gate, up = v[..., 0, :], v[..., 1, :]
        sg = 1 / (1 + torch.exp(-gate))
        return torch.stack([d * up * (sg + gate * sg * (1 - sg)), d * gate * sg], -2).flatten(-3)
    return dy


def _plain_linear(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    if c["train"]:
        dz = s["dy"].float() if s["z"] is None else _plain_dact(s["dy"].float(), s["z"].float(), c["act"])
        out = [(dz @ s["w"].float()).to(dt), (dz.t() @ s["x"].float()).to(dt)]
        return out + ([dz.sum(0).to(dt)] if c["bias"] else [])
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _plain_act(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(dt)


def _plain_grouped(s):
    """Every expert padded to the fullest one's rows: one batched product."""
    c = s["case"]
    dt, G, N, K, cap = _DT[c["dtype"]], c["G"], c["N"], c["K"], s["capacity"]
    r = torch.arange(c["rows"], device="cuda")
    e = torch.bucketize(r, s["m_offsets"][1:].long(), right=True)
    at = e * cap + r - s["m_offsets"].long()[e]
    w = s["w"].view(G, N, K).float()
    x = torch.zeros(G * cap, K, device="cuda").index_copy_(0, at, s["x"].float()).view(G, cap, K)
    if c["train"]:
        dz = s["dy"].float() if s["z"] is None else _plain_dact(s["dy"].float(), s["z"].float(), c["act"])
        dz = torch.zeros(G * cap, N, device="cuda").index_copy_(0, at, dz).view(G, cap, N)
        out = [torch.bmm(dz, w).view(G * cap, K)[at].to(dt), torch.bmm(dz.transpose(1, 2), x).view(G * N, K).to(dt)]
        return out + ([dz.sum(1).to(dt)] if c["bias"] else [])
    y = torch.bmm(x, w.transpose(1, 2)).view(G * cap, N)[at]
    if s["bias"] is not None:
        y = y + s["bias"].float()[e]
    return _plain_act(y, c["act"]).to(dt)


def _plain_scores(l, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    m = l.amax(1, keepdim=True)
    p = torch.exp(l - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p / p.sum(1, keepdim=True).clamp_min(1e-38)


def _plain_route(logits, k, scoring, bias, renormalize, scale):
    """(weights, experts, rows, m_offsets): the k highest-ranking experts of each token, the
    lower index first among equals; an expert whose logit is -inf is never chosen, and a
    choice that finds none left is -1 with weight 0.  Rows are numbered by expert, then by
    token; m_offsets[e] is expert e's first row."""
    l = logits.float()
    T, E = l.shape
    score = _plain_scores(l, scoring)
    rank = l if bias is None else (score + bias.float()).masked_fill(l == -math.inf, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :k]
    live = torch.gather(l, 1, order) != -math.inf
    w = torch.where(live, torch.gather(score, 1, order), torch.zeros((), device=l.device))
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    experts = torch.where(live, order, torch.full_like(order, -1))
    flat = torch.where(live, order, torch.full_like(order, E)).reshape(-1)
    by = torch.sort(flat, stable=True).indices
    rows = torch.empty_like(by).index_copy_(0, by, torch.arange(T * k, device=l.device))
    rows = torch.where(flat < E, rows, torch.full_like(rows, -1)).view(T, k)
    counts = (flat[:, None] == torch.arange(E, device=l.device)).sum(0)
    offsets = torch.cat([torch.zeros(1, dtype=counts.dtype, device=l.device), counts.cumsum(0)])
    return w * scale, experts.int(), rows.int(), offsets.int()


def _plain_route_backward(dw, logits, experts, scoring, renormalize, scale):
    l = logits.float()
    live = experts >= 0
    at = experts.long().clamp_min(0)
    score = _plain_scores(l, scoring)
    p = torch.where(live, torch.gather(score, 1, at), torch.zeros((), device=l.device))
    d = torch.where(live, dw, torch.zeros_like(dw)) * scale
    if renormalize:
        total = p.sum(1, keepdim=True)
        q = torch.where(total > 0, p / total, torch.zeros_like(p))
        d = torch.where(total > 0, (d - (q * d).sum(1, keepdim=True)) / total, torch.zeros_like(d))
    d = torch.where(live, d, torch.zeros_like(d))
    ds = torch.zeros_like(l).scatter_add_(1, at, d)
    if scoring == "sigmoid":
        dl = ds * score * (1 - score)
    else:
        dl = score * (ds - (score * ds).sum(1, keepdim=True))
    return dl.to(logits.dtype)


def _plain_move(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    weights, _, rows, _ = s["routing"]
    T, k = rows.shape
    live = (rows >= 0).reshape(-1)
    spare = T * k  # choices without a row write here
    at = torch.where(live, rows.reshape(-1).long(), torch.full((), spare, device=rows.device))
    read = rows.long().clamp_min(0)
    w = torch.where(rows >= 0, weights, torch.zeros_like(weights))

    def scatter(v):  # [T, k, K] -> expert order
        return torch.zeros(T * k + 1, c["K"], device=rows.device).index_copy_(0, at, v.reshape(T * k, -1))[:spare]

    gathered = scatter(s["x"].float()[:, None].expand(T, k, c["K"])).to(dt)
    er = torch.where((rows >= 0)[..., None], s["expert_rows"].float()[read], torch.zeros((), device=rows.device))
    y = (er * w[..., None]).sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = [gathered, y.to(dt)]
    if c["train"]:
        dy = s["dy"].float()
        dr = torch.where((rows >= 0)[..., None], s["drows"].float()[read], torch.zeros((), device=rows.device))
        out += [dr.sum(1).to(dt), scatter(dy[:, None] * w[..., None]).to(dt), (er * dy[:, None]).sum(2)]
    return out


# ----------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "linear":
            return _plain_linear(s)
        if op == "grouped":
            return _plain_grouped(s)
        if op == "move":
            return _plain_move(s)
        out = list(_plain_route(s["logits"], c["k"], c["scoring"], s["bias"], c["renormalize"], 1.0))
        if c["train"]:
            out.append(_plain_route_backward(s["dweights"], s["logits"], out[1], c["scoring"], c["renormalize"], 1.0))
        return out
    nv = _nv()
    if op == "linear":
        if c["train"]:
            out = nv.linear_backward(s["dy"], s["x"], s["w"], preact=s["z"], activation=c["act"], bias_grad=c["bias"])
            return [t for t in out if t is not None]
        return nv.linear(s["x"], s["w"], bias=s["bias"], activation=c["act"], residual=s["residual"])
    if op == "grouped":
        if c["train"]:
            out = nv.linear_grouped_backward(s["dy"], s["x"], s["w"], s["m_offsets"], preact=s["z"],
                                             activation=c["act"], bias_grad=c["bias"])
            return [t for t in out if t is not None]
        return nv.linear_grouped(s["x"], s["w"], s["m_offsets"], bias=s["bias"], activation=c["act"])
    if op == "route":
        r = nv.moe_route(s["logits"], c["k"], scoring=c["scoring"], bias=s["bias"], renormalize=c["renormalize"])
        out = [r.weights, r.experts, r.rows, r.m_offsets]
        if c["train"]:
            out.append(nv.moe_route_backward(s["dweights"], s["logits"], r, scoring=c["scoring"],
                                             renormalize=c["renormalize"]))
        return out
    r = nv.Routing(*s["routing"])
    out = [nv.moe_dispatch(s["x"], r), nv.moe_combine(s["expert_rows"], r, residual=s["residual"])]
    if c["train"]:
        out.append(nv.moe_dispatch_backward(s["drows"], r))
        out += nv.moe_combine_backward(s["dy"], s["expert_rows"], r)
    return out


def work(case):
    """Bytes: each input read once, each output written once.  Flops: the products."""
    op = case["op"]
    if op in ("linear", "grouped"):
        M = case["M"] if op == "linear" else case["rows"]
        # experts that have a row; the others' weights are not read
        G = 1 if op == "linear" else min(case["G"] - case["empty"], case["rows"])
        N, K = case["N"], case["K"]
        No = N // 2 if case["act"] == "swiglu" else N
        if case["train"]:
            all_groups = 1 if op == "linear" else case["G"]
            z = M * N if case["act"] != "none" else 0
            n = M * No + z + M * K + G * N * K + M * K + all_groups * N * (K + (1 if case["bias"] else 0))
            return {"bytes": 2 * n, "flops": 4 * M * N * K}
        n = M * K + G * N * (K + (1 if case["bias"] else 0)) + M * No * (2 if case.get("residual") else 1)
        return {"bytes": 2 * n, "flops": 2 * M * N * K}
    T, k = case["T"], case["k"]
    if op == "route":
        size, E = (4 if case["dtype"] == "fp32" else 2), case["E"]
        n = T * E * size + 12 * T * k + 4 * (E + 1) + (4 * E if case["select_bias"] else 0)
        if case["train"]:
            n += T * E * size + 4 * T * k
        return {"bytes": n, "flops": T * E * (3 + (4 if case["train"] else 0))}
    K = case["K"]
    n = 2 * K * (T + T * k) + 2 * K * (T * k + T * (2 if case["residual"] else 1)) + 8 * T * k
    f = 2 * T * k * K
    if case["train"]:
        n += 2 * K * (T * k + T) + 2 * K * (T + T * k) + 4 * T * k
        f += 4 * T * k * K
    return {"bytes": n, "flops": f}


# ----------------------------------------------------------------------------- 64 bits
def _act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act == "swiglu":
        M, N = z.shape
        v = z.reshape(M, N // 32, 32)
        return (v[:, :, :16] * torch.sigmoid(v[:, :, :16]) * v[:, :, 16:]).reshape(M, N // 2)
    return z


def _exact_products(case, s):
    """Expert by expert, gradients of the activation by autograd in 64 bits."""
    N, K, G = case["N"], case["K"], case.get("G", 1)
    cuts = s["cuts"] if case["op"] == "grouped" else [0, case["M"]]
    ys, dxs, dws, dbs = [], [], [], []
    for e in range(G):
        a, b = cuts[e], cuts[e + 1]
        x, w = s["x"][a:b].double(), s["w"][e * N:(e + 1) * N].double()
        if case["train"]:
            dz = s["dy"][a:b].double()
            if s["z"] is not None:
                z = s["z"][a:b].double().requires_grad_()
                with torch.enable_grad():
                    dz, = torch.autograd.grad(_act64(z, case["act"]), z, dz)
            dxs.append(dz @ w)
            dws.append(dz.t() @ x)
            dbs.append(dz.sum(0))
            continue
        y = x @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].double().reshape(-1, N)[e]
        y = _act64(y, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"][a:b].double()
        ys.append(y)
    if not case["train"]:
        return torch.cat(ys)
    out = [torch.cat(dxs), torch.cat(dws)]
    return out + ([dbs[0] if case["op"] == "linear" else torch.stack(dbs)] if case["bias"] else [])


def _choice(case, s):
    """The k experts of each token, one after another: the highest of the 32-bit ranking that
    is left, the lowest index among equals; -1 where only masked experts are left."""
    l = s["logits"].float()
    rank = l.clone()
    if s["bias"] is not None:
        rank = 1 / (1 + torch.exp(-l)) + s["bias"]
        rank[l == -math.inf] = -math.inf
    T, E = l.shape
    index = torch.arange(E, device="cuda").expand(T, E)
    chosen = torch.empty(T, case["k"], dtype=torch.int64, device="cuda")
    for j in range(case["k"]):
        top = rank.max(1, keepdim=True).values
        first = torch.where(rank == top, index, E).min(1, keepdim=True).values
        chosen[:, j:j + 1] = torch.where(top == -math.inf, -1, first)
        rank.scatter_(1, first, -math.inf)
    return chosen


def _exact_route(case, s):
    l = s["logits"].double().requires_grad_()
    dead = l.detach() == -math.inf
    with torch.enable_grad():
        if case["scoring"] == "sigmoid":
            score = torch.sigmoid(l)
        else:
            score = torch.softmax(l.masked_fill(dead.all(1, keepdim=True), 0.0), 1)
        chosen = _choice(case, s)
        p = torch.gather(score, 1, chosen.clamp_min(0)) * (chosen >= 0)
        if case["renormalize"]:
            total = p.sum(1, keepdim=True)
            p = p / torch.where(total > 0, total, torch.ones_like(total))
        out = [p.detach(), None, None, None]
        if case["train"]:
            dl, = torch.autograd.grad((p * s["dweights"].double()).sum(), l)
            out.append(torch.nan_to_num(dl))
    return out


def _exact_move(case, s):
    weights, _, rows, _ = s["routing"]
    T, k = rows.shape
    token = torch.arange(T, device="cuda")[:, None].expand(T, k)
    gathered = torch.zeros(T * k, case["K"], dtype=torch.float64, device="cuda")
    live = rows >= 0
    gathered[rows[live].long()] = s["x"].double()[token[live]]
    y = s["residual"].double().clone() if s["residual"] is not None else torch.zeros_like(s["x"], dtype=torch.float64)
    drows = torch.zeros_like(gathered)
    dx = torch.zeros_like(s["x"], dtype=torch.float64)
    dw = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        t = live[:, j].nonzero()[:, 0]
        r = rows[t, j].long()
        er, w = s["expert_rows"][r].double(), weights[t, j].double()[:, None]
        y[t] += er * w
        if case["train"]:
            dy = s["dy"][t].double()
            dx[t] += s["drows"][r].double()
            drows[r] = dy * w
            dw[t, j] = (er * dy).sum(1)
    return [gathered, y] + ([dx, drows, dw] if case["train"] else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "grouped"):
        return _exact_products(case, s)
    return _exact_route(case, s) if case["op"] == "route" else _exact_move(case, s)
