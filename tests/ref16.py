"""Plain 64-bit forms of the 16-bit linear and mixture-of-experts operators, with error
bounds derived from the formats: what the kernels' outputs may differ by.

Notation: u is the unit roundoff of the output type (bf16 2^-8, fp16 2^-11).  A product of
length K accumulated in fp32, 16 terms at a time, is off by at most
    acc(K) = (K / 16 + 16) 2^-22  times  sum |x_k w_k|
(each step's rounding or truncation is at most 2^-22 of the running magnitude, which the
sum of absolute products bounds; 16 for the steps inside a chunk and the final additions).
The activations have slopes below 1.2 and are computed to within 2^-19 relative.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half the smallest subnormal
ACTS = ("none", "relu", "silu", "gelu_tanh", "swiglu")


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act == "swiglu":
        v = z.reshape(z.shape[0], -1, 2, 16)
        return (v[:, :, 0] * torch.sigmoid(v[:, :, 0]) * v[:, :, 1]).reshape(z.shape[0], -1)
    return z


def act_bound(z, ez, act):
    """Bound of act's error for an error ez of z."""
    if act == "none":
        return ez
    if act == "swiglu":
        v, e = z.reshape(z.shape[0], -1, 2, 16), ez.reshape(z.shape[0], -1, 2, 16)
        g, up = v[:, :, 0], v[:, :, 1]
        silu = g * torch.sigmoid(g)
        out = 1.2 * e[:, :, 0] * (up.abs() + e[:, :, 1]) + silu.abs() * e[:, :, 1] + 2.0 ** -19 * (silu * up).abs()
        return out.reshape(z.shape[0], -1)
    return 1.2 * ez + 2.0 ** -19 * act64(z, act).abs()


def dact64(dy, z, act):
    if act == "none":
        return dy
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, act), z, dy)[0]


def acc(K):
    return (K / 16 + 16) * 2.0 ** -22


def groups_of(cuts):
    return [(g, cuts[g], cuts[g + 1]) for g in range(len(cuts) - 1)]


def forward64(x, w, cuts, bias, act, residual):
    """(y, bound of y's error before its rounding, z, bound of z) in 64 bits; zeros outside
    the groups."""
    G = len(cuts) - 1
    N, M = w.shape[0] // G, x.shape[0]
    No = N // 2 if act == "swiglu" else N
    y, ey = (torch.zeros(M, No, dtype=torch.float64, device=x.device) for _ in range(2))
    z, ez = (torch.zeros(M, N, dtype=torch.float64, device=x.device) for _ in range(2))
    for g, a, b in groups_of(cuts):
        if a == b:
            continue
        X, W = x[a:b].double(), w[g * N:(g + 1) * N].double()
        zz = X @ W.t()
        e = acc(X.shape[1]) * (X.abs() @ W.abs().t())
        if bias is not None:
            zz = zz + bias.double().reshape(G, N)[g]
            e = e + 2.0 ** -23 * zz.abs()
        yy, ee = act64(zz, act), act_bound(zz, e, act)
        if residual is not None:
            yy = yy + residual[a:b].double()
            ee = ee + 2.0 ** -23 * yy.abs()
        y[a:b], ey[a:b], z[a:b], ez[a:b] = yy, ee, zz, e
    return y, ey, z, ez


def backward64(dy, x, w, cuts, z, act):
    """[(dx, bound), (dw, bound), (db, bound)]: dZ is rounded to 16 bits before the products
    when there is an activation."""
    G = len(cuts) - 1
    N, (M, K) = w.shape[0] // G, x.shape
    u = U[x.dtype] if act != "none" else 0.0
    tiny = TINY[x.dtype] if act != "none" else 0.0
    out = [torch.zeros(s, dtype=torch.float64, device=x.device)
           for s in ((M, K), (M, K), (G * N, K), (G * N, K), (G, N), (G, N))]
    dx, edx, dw, edw, db, edb = out
    for g, a, b in groups_of(cuts):
        if a == b:
            continue
        X, W = x[a:b].double(), w[g * N:(g + 1) * N].double()
        dz = dact64(dy[a:b].double(), None if z is None else z[a:b].double(), act)
        # the derivative is computed to within 2^-18 of a value of at most |dy| times 1.2 (times
        # |gate| or |up| for SwiGLU, whose terms are below |z|_max in these tests)
        scale = dy[a:b].double().abs()
        if act == "swiglu":
            v = z[a:b].double().reshape(b - a, -1, 2, 16).abs() + 1.0
            scale = torch.stack([scale.reshape(b - a, -1, 16) * v[:, :, 1], scale.reshape(b - a, -1, 16) * v[:, :, 0]],
                                2).reshape(b - a, -1)
        e = (2.0 ** -18 * 1.2 * scale if act != "none" else torch.zeros_like(dz))
        ez = u * dz.abs() + tiny + e
        dx[a:b], edx[a:b] = dz @ W, acc(N) * ((dz.abs() + ez) @ W.abs()) + ez @ W.abs()
        s = slice(g * N, (g + 1) * N)
        dw[s], edw[s] = dz.t() @ X, acc(b - a) * ((dz.abs() + ez).t() @ X.abs()) + ez.t() @ X.abs()
        db[g], edb[g] = dz.sum(0), ((b - a) * 2.0 ** -24 * dz.abs() + e).sum(0)
    return [(dx, edx), (dw, edw), (db, edb)]


def assert_close(got, ref, bound, what=""):
    """got is ref + (error within bound), rounded once to got's type."""
    u, tiny = U[got.dtype], TINY[got.dtype]
    limit = bound + u * (ref.abs() + bound) + tiny
    err = (got.double() - ref).abs()
    bad = ~(err <= limit)
    if bad.any():
        i = int((err - limit).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds; worst at {i}: "
                             f"{got.flatten()[i].item()} for {ref.flatten()[i].item()}, "
                             f"limit {limit.flatten()[i].item():.3e}")


def route64(logits, k, scoring, bias, renormalize, scale):
    """(weights 64-bit, experts, rows, offsets) by a plain loop over tokens, on the CPU.  The
    choice ranks the 32-bit scores when there is a bias, as the operator does."""
    l32 = logits.float().cpu()
    T, E = l32.shape
    l = l32.double()
    experts = torch.full((T, k), -1, dtype=torch.int32)
    weights = torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        live = [e for e in range(E) if l32[t, e] > -float("inf")]
        if bias is None:
            rank = l32[t]
        else:
            rank = 1 / (1 + torch.exp(-logits[t].float())).cpu() + bias.cpu()
        chosen = sorted(live, key=lambda e: (-rank[e].item(), e))[:k]
        if scoring == "sigmoid":
            score = torch.sigmoid(l[t])
        else:
            score = torch.zeros(E, dtype=torch.float64)
            if live:
                score[live] = torch.softmax(l[t, live], 0)
        w = [score[e].item() for e in chosen]
        total = sum(w) if renormalize else 1.0
        for j, e in enumerate(chosen):
            experts[t, j] = e
            weights[t, j] = w[j] / total * scale if total else 0.0
    offsets = [0]
    rows = torch.full((T, k), -1, dtype=torch.int32)
    for e in range(E):
        r = offsets[-1]
        for t, j in (experts == e).nonzero().tolist():
            rows[t, j] = r
            r += 1
        offsets.append(r)
    return weights, experts, rows, torch.tensor(offsets, dtype=torch.int32)
