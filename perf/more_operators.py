"""The operators between token ids and log probabilities, as cases to measure.

The 16-bit layers and the experts of an NVFP4 model stand between two ends that share the
vocabulary, and a decode step passes its few tokens through the experts one by one.  Three
operators close that path:

  embedding  rows of a 16-bit table by token id, scaled; and the table's gradient, by sorted
             tokens
  experts    a whole mixture-of-experts layer of a few tokens from its router's logits: choice,
             SwiGLU experts, weighted sum, residual
  logprobs   log probability of given tokens, entropy and the most probable alternatives of
             rows of logits; and the gradient of the logits

Each case runs in a plain form (elementary torch operations in 32 bits, rounded once at the
end) or, where `own` is true, through the nvfp4_b200 package.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


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
        # the lookup that opens a decode step of a small batch: latency
        dict(name="embedding decode 16", op="embedding", train=False, T=16, V=131072, K=4096, scaled=False, padded=0.0,
             dtype="bf16"),
        # a packed prompt with padding tokens, an odd vocabulary and rows that fill no power of two
        dict(name="embedding prompt", op="embedding", train=False, T=8191, V=50257, K=4104, scaled=True, padded=0.1,
             dtype="fp16"),
        # training step: the gradient of a large table, most of whose rows no token touches
        dict(name="embedding train", op="embedding", train=True, T=16384, V=131072, K=4096, scaled=False, padded=0.0,
             dtype="bf16"),
        # training step of a small vocabulary over many tokens: long runs of the same token
        dict(name="embedding train small table", op="embedding", train=True, T=65533, V=32000, K=2048, scaled=True,
             padded=0.03, dtype="fp16"),
        # one token through 8 of 128 small experts: the latency of a decode step
        dict(name="experts 1 token", op="experts", T=1, E=128, k=8, K=2048, F=768, scoring="softmax",
             select_bias=False, renormalize=True, residual=True, masked=0.0, dtype="bf16", logits="bf16"),
        # a small batch through 64 experts with a balancing bias, sizes that fill no tile
        dict(name="experts 13 tokens", op="experts", T=13, E=64, k=6, K=2056, F=1408, scoring="sigmoid",
             select_bias=True, renormalize=True, residual=False, masked=0.05, dtype="fp16", logits="fp32"),
        # a batch through all of 8 large experts: the weights' bytes
        dict(name="experts 32 tokens", op="experts", T=32, E=8, k=2, K=4096, F=14336, scoring="softmax",
             select_bias=False, renormalize=True, residual=True, masked=0.0, dtype="bf16", logits="bf16"),
        # one sampled token, its log probability and five alternatives: latency
        dict(name="logprobs 1 token", op="logprobs", train=False, T=1, V=50257, W=50264, top=5, entropy=False,
             temperature=1.0, masked=0.0, ignored=0.0, dtype="fp32"),
        # a decode batch under constrained sampling: most of the vocabulary masked
        dict(name="logprobs decode 16", op="logprobs", train=False, T=16, V=131072, W=131072, top=20, entropy=True,
             temperature=0.7, masked=0.6, ignored=0.0, dtype="bf16"),
        # scoring a long prompt with alternatives
        dict(name="logprobs prompt", op="logprobs", train=False, T=4096, V=131072, W=131072, top=8, entropy=True,
             temperature=1.0, masked=0.0, ignored=0.05, dtype="bf16"),
        # training step with an entropy term, an odd vocabulary in padded rows
        dict(name="logprobs train", op="logprobs", train=True, T=4093, V=100003, W=100032, top=0, entropy=True,
             temperature=1.0, masked=0.0, ignored=0.2, dtype="bf16"),
        # training step on 32-bit logits of a small vocabulary
        dict(name="logprobs train fp32", op="logprobs", train=True, T=2047, V=32000, W=32000, top=0, entropy=False,
             temperature=0.9, masked=0.0, ignored=0.0, dtype="fp32"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _largest():
    """Bytes of the largest listed case of each operator."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), work(c)["bytes"])
    return most


def draw(rng):
    op = rng.choice(["embedding", "experts", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if op == "embedding":
            case = dict(op=op, train=rng.random() < 0.5, T=_log_int(rng, 1, 65536), V=_log_int(rng, 256, 262144),
                        K=_log_int(rng, 64, 8192, 8), scaled=rng.random() < 0.5, padded=rng.choice([0.0, 0.0, 0.1]),
                        dtype=dtype)
        elif op == "experts":
            E = rng.choice([8, 16, 60, 64, 128, 160, 256])
            scoring = rng.choice(["softmax", "sigmoid"])
            case = dict(op=op, T=_log_int(rng, 1, 64), E=E, k=rng.randint(1, 8), K=_log_int(rng, 256, 7168, 8),
                        F=_log_int(rng, 128, 14336, 16), scoring=scoring,
                        select_bias=scoring == "sigmoid" and rng.random() < 0.5, renormalize=rng.random() < 0.7,
                        residual=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.05]), dtype=dtype,
                        logits=rng.choice([dtype, "fp32"]))
            # all experts' weights and 32-bit copies of those in use fit beside the other passes'
            if E * case["F"] * case["K"] * 3 > 3 * 8 * 14336 * 4096:
                continue
        else:
            V = _log_int(rng, 1000, 262144)
            case = dict(op=op, train=rng.random() < 0.5, T=_log_int(rng, 1, 16384), V=V,
                        W=V if rng.random() < 0.4 else (V + 63) // 64 * 64, top=rng.choice([0, 1, 5, 20, 32]),
                        entropy=rng.random() < 0.5, temperature=rng.choice([1.0, 0.7, 1.3]),
                        masked=rng.choice([0.0, 0.0, 0.5]), ignored=rng.choice([0.0, 0.1]),
                        dtype=rng.choice(["bf16", "fp16", "fp32"]))
            if case["train"]:
                case["top"] = 0
        if work(case)["bytes"] <= _largest()[op]:
            return case


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _weight(g, rows, K, dtype, scale):
    w = torch.empty(rows, K, device="cuda", dtype=dtype)
    step = max(1, (1 << 27) // K)
    for r in range(0, rows, step):
        part = w[r:r + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(scale))
    return w


def _uniform(g, *shape):
    return torch.rand(shape, device="cuda", generator=g)


def _tokens(g, T, V):
    """Token ids of text: the n-th commonest about n times rarer than the first, the common
    ones spread over the vocabulary."""
    rank = (float(V + 1) ** _uniform(g, T).double()).long() - 1
    return rank.clamp_(0, V - 1) * 7919 % V


def prepare(case, seed):
    g = _gen(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    s = dict(case=case)
    if op == "embedding":
        T, V, K = case["T"], case["V"], case["K"]
        t = _tokens(g, T, V)
        s["tokens"] = torch.where(_uniform(g, T) < case["padded"], torch.full_like(t, -1), t)
        s["scale"] = math.sqrt(K) if case["scaled"] else 1.0
        if case["train"]:
            s["dy"] = _normal(g, (T, K), dt)
        else:
            s["table"] = _weight(g, V, K, dt, 0.02 if case["scaled"] else 1.0)
    elif op == "experts":
        T, E, K, F = case["T"], case["E"], case["K"], case["F"]
        s["x"] = _normal(g, (T, K), dt)
        s["w13"] = _weight(g, E * 2 * F, K, dt, K ** -0.5)
        s["w2"] = _weight(g, E * K, F, dt, F ** -0.5)
        l = torch.randn(T, E, device="cuda", generator=g) * 2
        if case["masked"]:
            l.masked_fill_(_uniform(g, T, E) < case["masked"], -math.inf)
            l.masked_fill_(_uniform(g, T, 1) < case["masked"], -math.inf)  # padding tokens
        s["logits"] = l.to(_DT[case["logits"]])
        s["bias"] = torch.randn(E, device="cuda", generator=g) * 0.05 if case["select_bias"] else None
        s["residual"] = _normal(g, (T, K), dt) if case["residual"] else None
    else:
        T, V, W = case["T"], case["V"], case["W"]
        l = torch.empty(T, W, device="cuda", dtype=dt)
        target = torch.empty(T, device="cuda", dtype=torch.int64)
        step = max(1, (1 << 27) // W)
        for r in range(0, T, step):
            part = torch.randn(l[r:r + step].shape, device="cuda", generator=g).mul_(2.5)
            part += 0.05 * part * part  # a longer upper tail: some tokens stand out
            n = part.shape[0]
            t = (_uniform(g, n) * V).long().clamp_(max=V - 1)
            target[r:r + step] = t
            if case["masked"]:
                part.masked_fill_(_uniform(g, n, W) < case["masked"], -math.inf)
                part.scatter_(1, t[:, None], 4.0)
            l[r:r + step].copy_(part)
        s["logits"] = l
        s["targets"] = torch.where(_uniform(g, T) < case["ignored"], torch.full_like(target, -100), target)
        if case["train"]:
            s["dlogprobs"] = torch.randn(T, device="cuda", generator=g) / T
            s["dentropy"] = torch.randn(T, device="cuda", generator=g) / T if case["entropy"] else None
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_embedding(s):
    c = s["case"]
    dt, V, K = _DT[c["dtype"]], c["V"], c["K"]
    live = (s["tokens"] >= 0) & (s["tokens"] < V)
    at = torch.where(live, s["tokens"], torch.zeros_like(s["tokens"]))
    if c["train"]:
        spare = torch.where(live, at, torch.full_like(at, V))  # tokens without a row add up past the table
        d = torch.zeros(V + 1, K, device="cuda").index_add_(0, spare, s["dy"].float())
        return (d[:V] * s["scale"]).to(dt)
    y = s["table"][at].float() * s["scale"]
    return torch.where(live[:, None], y, torch.zeros((), device="cuda")).to(dt)


def _plain_scores(l, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    m = l.amax(1, keepdim=True)
    p = torch.exp(l - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p / p.sum(1, keepdim=True).clamp_min(1e-38)


def _plain_choice(s):
    """(weights, experts) of each token: the k highest-ranking experts, the lowest index first
    among equals; -1 and weight 0 where only masked experts are left."""
    c = s["case"]
    l = s["logits"].float()
    score = _plain_scores(l, c["scoring"])
    rank = l if s["bias"] is None else (score + s["bias"]).masked_fill(l == -math.inf, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    live = torch.gather(l, 1, order) != -math.inf
    w = torch.where(live, torch.gather(score, 1, order), torch.zeros((), device=l.device))
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return w, torch.where(live, order, torch.full_like(order, -1))


def _plain_swiglu(z):
    v = z.unflatten(-1, (-1, 2, 16))  # blocks of 16 gate columns, then 16 up columns
    gate, up = v[..., 0, :], v[..., 1, :]
    return (gate / (1 + torch.exp(-gate)) * up).flatten(-2)


def _plain_experts(s):
    """Fewer choices than experts: the weights of each choice, gathered.  Otherwise every token
    through every expert, with weight zero where it was not chosen."""
    c = s["case"]
    T, E, k, K, F = c["T"], c["E"], c["k"], c["K"], c["F"]
    w, experts = _plain_choice(s)
    x = s["x"].float()
    w13, w2 = s["w13"].view(E, 2 * F, K), s["w2"].view(E, K, F)
    if T * k < E:
        at = experts.clamp_min(0).reshape(-1)
        z = torch.bmm(w13[at].float(), x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
        y = torch.bmm(w2[at].float(), _plain_swiglu(z)[:, :, None]).view(T, k, K)
        y = (y * w[:, :, None]).sum(1)
    else:
        by = torch.zeros(T, E, device="cuda").scatter_add_(1, experts.clamp_min(0), w)
        y = torch.zeros(T, K, device="cuda")
        step = max(1, (1 << 30) // (2 * F * K))
        for e in range(0, E, step):
            z = torch.matmul(x, w13[e:e + step].float().transpose(1, 2))
            o = torch.bmm(_plain_swiglu(z), w2[e:e + step].float().transpose(1, 2))
            y += (o * by[:, e:e + step].t()[:, :, None]).sum(0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(_DT[c["dtype"]])


def _plain_logprobs(s):
    """Log probabilities of the targets (0 for one outside the vocabulary), entropy, the top
    alternatives (the lowest index first among equals); masked tokens have logit -inf."""
    c = s["case"]
    V = c["V"]
    raw = s["logits"][:, :V].float()
    l = raw / c["temperature"]
    m = l.amax(1, keepdim=True)
    e = torch.exp(l - m)
    lse = m + torch.log(e.sum(1, keepdim=True))
    live = (s["targets"] >= 0) & (s["targets"] < V)
    at = torch.where(live, s["targets"], torch.zeros_like(s["targets"]))
    zero = torch.zeros((), device="cuda")
    logp = torch.where(live, (torch.gather(l, 1, at[:, None]) - lse)[:, 0], zero)
    out = [logp]
    entropy = None
    if c["entropy"]:
        p = torch.exp(l - lse)
        entropy = -torch.where(p > 0, p * (l - lse), zero).sum(1)
        out.append(entropy)
    if c["top"]:
        index = torch.arange(V, device="cuda", dtype=torch.int32)
        values, tokens = [], []
        rest = raw.clone()
        for _ in range(c["top"]):
            v = rest.amax(1, keepdim=True)
            first = torch.where(rest == v, index, V).amin(1, keepdim=True)
            values.append(v)
            tokens.append(first)
            rest.scatter_(1, first.long(), -math.inf)
        values, tokens = torch.cat(values, 1), torch.cat(tokens, 1)
        out += [values / c["temperature"] - lse, torch.where(values > -math.inf, tokens, -1)]
    if c["train"]:
        p = torch.exp(l - lse)
        g = torch.where(live, s["dlogprobs"], zero)[:, None]
        d = -g * p
        if entropy is not None:
            d = d - s["dentropy"][:, None] * torch.where(p > 0, p * (l - lse + entropy[:, None]), zero)
        d.scatter_add_(1, at[:, None], g)
        d = (d / c["temperature"]).masked_fill(raw == -math.inf, 0.0)
        full = torch.zeros(c["T"], c["W"], device="cuda", dtype=s["logits"].dtype)
        full[:, :V] = d.to(full.dtype)
        out.append(full)
    return out


# ----------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"embedding": _plain_embedding, "experts": _plain_experts, "logprobs": _plain_logprobs}[op](s)
    nv = _nv()
    if op == "embedding":
        if c["train"]:
            return nv.embedding_backward(s["dy"], s["tokens"], c["V"], scale=s["scale"])
        return nv.embedding(s["tokens"], s["table"], scale=s["scale"])
    if op == "experts":
        return nv.moe_layer(s["x"], s["logits"], s["w13"], s["w2"], c["k"], scoring=c["scoring"], bias=s["bias"],
                            renormalize=c["renormalize"], residual=s["residual"])
    r = nv.token_logprobs(s["logits"], s["targets"], vocab=c["V"], top_k=c["top"], temperature=c["temperature"],
                          entropy=c["entropy"])
    out = [r.logprobs]
    if c["entropy"]:
        out.append(r.entropy)
    if c["top"]:
        out += [r.top_logprobs, r.top_tokens]
    if c["train"]:
        out.append(nv.token_logprobs_backward(s["dlogprobs"], s["logits"], s["targets"], r, dentropy=s["dentropy"],
                                              vocab=c["V"], temperature=c["temperature"]))
    return out


def _active(case):
    """Experts that T x k random choices are expected to touch."""
    E, k = case["E"], case["k"]
    return E * (1.0 - (1.0 - k / E) ** case["T"])


def work(case):
    """Bytes: each input read once, each output written once.  Flops: sums and products."""
    op = case["op"]
    if op == "embedding":
        T, V, K = case["T"], case["V"], case["K"]
        if case["train"]:
            return {"bytes": 8 * T + 2 * T * K + 2 * V * K, "flops": 2 * T * K}
        return {"bytes": 8 * T + 2 * min(T, V) * K + 2 * T * K, "flops": T * K}
    if op == "experts":
        T, K, F = case["T"], case["K"], case["F"]
        size = 4 if case["logits"] == "fp32" else 2
        weights = int(_active(case) * 3 * F * K)
        return {"bytes": 2 * weights + T * case["E"] * size + 2 * T * K * (3 if case["residual"] else 2),
                "flops": 6 * T * case["k"] * F * K}
    T, V = case["T"], case["V"]
    size = 4 if case["dtype"] == "fp32" else 2
    n = T * V * size + 12 * T + 8 * T * case["top"] + (4 * T if case["entropy"] else 0)
    if case["train"]:
        n += T * case["W"] * size + 4 * T * (2 if case["entropy"] else 1)
    return {"bytes": n, "flops": T * V * ((8 if case["entropy"] else 5) + (6 if case["train"] else 0))}


# ----------------------------------------------------------------------------- 64 bits
def _exact_embedding(case, s):
    t = s["tokens"]
    known = (t >= 0) & (t < case["V"])
    if case["train"]:
        d = torch.zeros(case["V"], case["K"], dtype=torch.float64, device="cuda")
        return d.index_put_((t[known],), s["dy"][known].double() * s["scale"], accumulate=True)
    y = torch.zeros(case["T"], case["K"], dtype=torch.float64, device="cuda")
    y[known] = s["table"][t[known]].double() * s["scale"]
    return y


def _exact_experts(case, s):
    """Token by token choice in 32-bit ranks, then expert by expert in 64 bits."""
    T, E, K, F = case["T"], case["E"], case["K"], case["F"]
    l = s["logits"].float()
    rank = l.clone()
    if s["bias"] is not None:
        rank = 1 / (1 + torch.exp(-l)) + s["bias"]
        rank[l == -math.inf] = -math.inf
    rank, l = rank.cpu().tolist(), l.double().cpu()
    y = s["residual"].double().clone() if s["residual"] is not None else torch.zeros(T, K, dtype=torch.float64,
                                                                                     device="cuda")
    rows = {}
    for t in range(T):
        free = [e for e in range(E) if rank[t][e] != -math.inf]
        chosen = sorted(free, key=lambda e: (-rank[t][e], e))[:case["k"]]
        if not chosen:
            continue
        p = torch.sigmoid(l[t]) if case["scoring"] == "sigmoid" else torch.softmax(l[t], 0)
        total = sum(p[e].item() for e in chosen) if case["renormalize"] else 1.0
        for e in chosen:
            rows.setdefault(e, []).append((t, p[e].item() / total))
    for e, members in sorted(rows.items()):
        t = torch.tensor([m[0] for m in members], device="cuda")
        w = torch.tensor([m[1] for m in members], device="cuda", dtype=torch.float64)
        z = (s["x"][t].double() @ s["w13"][e * 2 * F:(e + 1) * 2 * F].double().t()).view(len(members), F // 16, 32)
        h = torch.nn.functional.silu(z[:, :, :16]) * z[:, :, 16:]
        y[t] += w[:, None] * (h.reshape(len(members), F) @ s["w2"][e * K:(e + 1) * K].double().t())
    return y


def _exact_logprobs(case, s):
    T, V = case["T"], case["V"]
    parts = []
    step = max(1, (1 << 26) // V)
    for r in range(0, T, step):
        l = s["logits"][r:r + step, :V].double().requires_grad_(case["train"])
        with torch.enable_grad():
            lp = torch.log_softmax(l / case["temperature"], 1)
            t = s["targets"][r:r + step]
            known = (t >= 0) & (t < V)
            mine = lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
            mine = torch.where(known, mine, torch.zeros_like(mine))
            out = [mine.detach()]
            loss = (mine * s["dlogprobs"][r:r + step].double()).sum() if case["train"] else None
            if case["entropy"]:
                h = -(lp.exp() * lp.masked_fill(lp == -math.inf, 0.0)).sum(1)
                out.append(h.detach())
                if case["train"]:
                    loss = loss + (h * s["dentropy"][r:r + step].double()).sum()
        if case["top"]:
            out += [lp.detach().topk(case["top"], 1).values, None]
        if case["train"]:
            d, = torch.autograd.grad(loss, l)
            d = d.masked_fill(l.detach() == -math.inf, 0.0)
            out.append(torch.nn.functional.pad(d, (0, case["W"] - V)))
        parts.append(out)
    return [None if column[0] is None else torch.cat(column) for column in zip(*parts)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"embedding": _exact_embedding, "experts": _exact_experts, "logprobs": _exact_logprobs}[case["op"]](case, s)
