"""GPU: the whole mixture-of-experts layer of a few tokens against a plain 64-bit form, and as
a part of a decode step."""
import importlib.util
import math
import os

import pytest
import torch

import ref16 as R

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def layer(T, E, K, F, dtype, seed, residual=True, logits=torch.float32):
    g = gen(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    return dict(x=normal(T, K), logits=(torch.randn(T, E, device="cuda", generator=g) * 2).to(logits),
                w13=normal(E * 2 * F, K, scale=K ** -0.5), w2=normal(E * K, F, scale=F ** -0.5),
                residual=normal(T, K) if residual else None)


def layer64(x, logits, w13, w2, k, scoring, bias, renormalize, scale, residual, rounded_rows=False):
    """(y, bound).  The hidden state is rounded to 16 bits; the weights are a few fp32 operations
    (within 1e-5); the sum of k products is fp32.  rounded_rows: each expert's result is rounded
    too, as for more than a few tokens."""
    (T, K), E, F, u = x.shape, logits.shape[1], w2.shape[1], R.U[x.dtype]
    weights, experts, _, _ = R.route64(logits, k, scoring, bias, renormalize, scale)
    y = torch.zeros(T, K, dtype=torch.float64, device="cuda") if residual is None else residual.double()
    b = 2.0 ** -23 * y.abs()
    for e in range(E):
        t, j = (experts == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        w = weights[t, j].cuda()[:, None]
        X, A, B = x[t.cuda()].double(), w13[e * 2 * F:(e + 1) * 2 * F].double(), w2[e * K:(e + 1) * K].double()
        z = X @ A.t()
        ez = R.acc(K) * (X.abs() @ A.abs().t())
        h, eh = R.act64(z, "swiglu"), R.act_bound(z, ez, "swiglu")
        eh = eh + u * (h.abs() + eh) + R.TINY[x.dtype]
        o = h @ B.t()
        eo = R.acc(F) * ((h.abs() + eh) @ B.abs().t()) + eh @ B.abs().t()
        if rounded_rows:
            eo = eo + u * (o.abs() + eo) + R.TINY[x.dtype]
        y.index_add_(0, t.cuda(), w * o)
        b.index_add_(0, t.cuda(), w.abs() * (eo + (1e-5 + 2.0 ** -22) * o.abs()))
    return y, b + 2.0 ** -22 * y.abs()


def check(nv, d, k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    args = d["x"], d["logits"], d["w13"], d["w2"], k
    y = nv.moe_layer(*args, scoring=scoring, bias=bias, renormalize=renormalize, scale=scale, residual=d["residual"])
    torch.cuda.synchronize()
    nv.device_status()
    more = d["x"].shape[0] > nv.moe.FEW_TOKENS
    ref, bound = layer64(*args, scoring, bias, renormalize, scale, d["residual"], rounded_rows=more)
    R.assert_close(y, ref, bound)
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,K,F", [
    (1, 1, 1, 8, 16), (1, 8, 2, 64, 48), (2, 3, 1, 24, 1040), (3, 4, 4, 72, 16), (8, 128, 8, 2048, 768),
    (9, 5, 1, 2056, 2064), (12, 40, 32, 40, 32), (16, 1, 1, 2048, 2048), (14, 2, 2, 1032, 1024), (13, 64, 6, 264, 80),
    (16, 256, 8, 1024, 64), (17, 2, 2, 1032, 1024), (25, 6, 3, 4104, 32), (32, 8, 2, 512, 1408), (33, 3, 3, 2056, 1040),
    (49, 256, 8, 1024, 48), (64, 1, 1, 2048, 512), (64, 4, 2, 520, 96), (64, 40, 32, 40, 32), (64, 256, 4, 512, 256),
    (18, 1, 1, 8, 16), (30, 4, 3, 128, 64), (48, 8, 8, 136, 5008), (61, 16, 8, 2056, 1424), (64, 8, 1, 8200, 1040),
    (64, 2, 1, 1 << 17, 16), (20, 3, 2, 64, 1 << 15)])
def test_moe_layer(nv, cuda_dev, T, E, k, K, F, dtype):
    """One tile of rows to four units' sixteens, sizes that fill no chunk, stage or tile, more warps
    than chunks, fewer slots than pieces, tiles cut into many parts, experts without a token."""
    check(nv, layer(T, E, K, F, dtype, T + E, residual=T % 2 == 1, logits=dtype if T % 3 else torch.float32), k)


@pytest.mark.parametrize("scoring,bias,renorm,scale", [("softmax", False, False, 1.0), ("sigmoid", False, True, 2.5),
                                                       ("sigmoid", True, True, 1.0), ("sigmoid", True, False, 0.5)])
def test_moe_layer_scores(nv, cuda_dev, scoring, bias, renorm, scale):
    d = layer(11, 40, 256, 160, torch.bfloat16, 3)
    b = torch.randn(40, device="cuda", generator=gen(1)) * 0.1 if bias else None
    check(nv, d, 5, scoring, b, renorm, scale)


@pytest.mark.parametrize("T", [10, 41])
@pytest.mark.parametrize("K,F", [(64, 32), (72, 48), (2048, 1024)])
def test_moe_layer_masks(nv, cuda_dev, K, F, T):
    """Masked experts (-inf, NaN, the lowest value), tokens with fewer experts left than they
    choose, with none, and a batch of such tokens alone."""
    d = layer(T, 6, K, F, torch.bfloat16, 5)
    d["logits"][0] = -math.inf
    d["logits"][1, 1:] = -math.inf
    d["logits"][2, ::2] = math.nan
    d["logits"][3] = torch.finfo(torch.float32).min
    d["logits"][4, :5] = torch.finfo(torch.float32).min
    d["logits"][9] = math.nan
    clean = dict(d, logits=torch.where(d["logits"].isnan(), torch.full_like(d["logits"], -math.inf), d["logits"]))
    y = check(nv, clean, 3)
    assert torch.equal(y, nv.moe_layer(d["x"], d["logits"], d["w13"], d["w2"], 3, residual=d["residual"]))
    assert torch.equal(y[0], d["residual"][0]) and torch.equal(y[9], d["residual"][9])
    d["logits"][:] = -math.inf
    assert torch.equal(check(nv, d, 3), d["residual"])
    assert not check(nv, dict(d, residual=None), 2).any()


@pytest.mark.parametrize("T", [4, 35])
def test_moe_layer_reads_chosen_experts_only(nv, cuda_dev, T):
    """Weights of experts that no token chose, and rows beside the tokens', may hold anything; an
    infinity in one token's row stays in its own result."""
    E, K, F = 8, 136, 48
    d = layer(T, E, K, F, torch.float16, 2)
    d["logits"][:, 4:] = -math.inf
    want = check(nv, d, 2)
    for w, rows in (("w13", 2 * F), ("w2", K)):
        d[w].view(E, rows, -1)[4:] = math.nan
    wide = torch.full((T + 2, K + 24), math.inf, device="cuda", dtype=torch.float16)
    wide[1:T + 1, 8:8 + K] = d["x"]
    d["x"] = wide[1:T + 1, 8:8 + K]
    got = nv.moe_layer(d["x"], d["logits"], d["w13"], d["w2"], 2, residual=d["residual"])
    assert torch.equal(got, want)
    d["x"][2] = math.inf
    got = nv.moe_layer(d["x"], d["logits"], d["w13"], d["w2"], 2, residual=d["residual"])
    assert got[2].isnan().all() and torch.equal(got[:2], want[:2]) and torch.equal(got[3:], want[3:])


def test_moe_layer_one_expert_for_all(nv, cuda_dev):
    """Every token to the same expert: the most rows an expert can have."""
    for T in (7, 8, 9, 16, 17, 24, 33, 57, 64):
        d = layer(T, 5, 512, 96, torch.bfloat16, T)
        d["logits"][:, 3] = 50.0
        check(nv, d, 1)
        check(nv, d, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_layer_uneven_rows(nv, cuda_dev, dtype):
    """Few rows an expert on average and most of them one expert's: units of up to four sixteens,
    beside experts of one row, with whole and partial stages."""
    for T in (9, 16, 17, 32, 33, 50, 64):
        d = layer(T, 64, 1032, 1040, dtype, T, residual=T % 2 == 0)
        d["logits"][:, 3] = 50.0
        check(nv, d, 1)
        check(nv, d, 3)


def test_moe_layer_same_bits(nv, cuda_dev):
    d = layer(50, 10, 1032, 528, torch.bfloat16, 1)
    args = d["x"], d["logits"], d["w13"], d["w2"], 4
    y = nv.moe_layer(*args, residual=d["residual"])
    for _ in range(20):
        assert torch.equal(y, nv.moe_layer(*args, residual=d["residual"]))


def test_moe_layer_same_bits_and_agreement(nv, cuda_dev):
    d = layer(16, 32, 2048, 1024, torch.bfloat16, 1)
    args = d["x"], d["logits"], d["w13"], d["w2"], 4
    y = nv.moe_layer(*args, residual=d["residual"])
    for _ in range(20):
        assert torch.equal(y, nv.moe_layer(*args, residual=d["residual"]))
    # the rows of a batch are those of each token alone, up to the sums' different order: none,
    # since a unit's split depends on the weights' sizes alone
    for t in (0, 7, 15):
        one = nv.moe_layer(d["x"][t:t + 1], d["logits"][t:t + 1], d["w13"], d["w2"], 4, residual=d["residual"][t:t + 1])
        assert torch.equal(one[0], y[t])


@pytest.mark.parametrize("T", [0, 65, 128, 200])
def test_moe_layer_more_tokens(nv, cuda_dev, T):
    d = layer(T, 8, 256, 96, torch.bfloat16, 4)
    if T == 0:
        assert nv.moe_layer(d["x"], d["logits"], d["w13"], d["w2"], 2).shape == (0, 256)
        return
    check(nv, d, 2)
    check(nv, dict(d, residual=None), 3, "sigmoid")


@pytest.mark.parametrize("A,B,E", [(8, 5, 16), (40, 64, 16), (50, 25, 8)])
def test_moe_layer_streams_and_graphs(nv, cuda_dev, A, B, E):
    """Calls on two streams at once, and two captured graphs whose replays overlap."""
    a, b = layer(A, E, 1024, 512, torch.bfloat16, 1), layer(B, E, 1024, 512, torch.bfloat16, 2)

    def call(d):
        return nv.moe_layer(d["x"], d["logits"], d["w13"], d["w2"], 4, residual=d["residual"])

    want = [call(a).clone(), call(b).clone()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, d in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(d))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    graphs, out = [], []
    for d in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(call(d))
        graphs.append(g)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out))
    a["logits"].copy_(b["logits"].flip(0).repeat(2, 1)[:A])  # replays follow inputs changed in place
    graphs[0].replay()
    assert torch.equal(out[0], call(a))
    nv.device_status()


def test_moe_layer_refusals(nv, cuda_dev):
    d = layer(4, 8, 64, 32, torch.bfloat16, 1)
    x, l, w13, w2 = d["x"], d["logits"], d["w13"], d["w2"]
    for call in (lambda: nv.moe_layer(x.float(), l, w13, w2, 2), lambda: nv.moe_layer(x.cpu(), l, w13, w2, 2),
                 lambda: nv.moe_layer(x[:, :60], l, w13, w2, 2), lambda: nv.moe_layer(x, l[:3], w13, w2, 2),
                 lambda: nv.moe_layer(x, l, w13[:-1], w2, 2), lambda: nv.moe_layer(x, l, w13, w2[:-1], 2),
                 lambda: nv.moe_layer(x, l, w13.half(), w2, 2), lambda: nv.moe_layer(x, l, w13, w2[:, :24], 2),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, scoring="none"),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, bias=torch.zeros(8, device="cuda")),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, residual=x[:2]),
                 lambda: nv.moe_layer(x, l.double(), w13, w2, 2)):
        with pytest.raises(ValueError):
            call()
    for k in (0, 9):
        with pytest.raises(nv.NVFP4Error):
            nv.moe_layer(x, l, w13, w2, k)


def test_decode_step(nv, cuda_dev):
    """The operators together, as a decode step and its scoring use them: embedding, router,
    experts, output projection by the same table, log probabilities."""
    rows, K, F, E = 1000, 256, 128, 16
    g = gen(7)
    table = (torch.randn(rows, K, device="cuda", generator=g) * K ** -0.5).bfloat16()
    router = (torch.randn(E, K, device="cuda", generator=g)).bfloat16()
    d = layer(6, E, K, F, torch.bfloat16, 8)
    tokens = torch.tensor([3, 999, -1, 0, 3, 500], device="cuda")
    x = nv.embedding(tokens, table, K ** 0.5)
    d["x"] = d["residual"] = x
    d["logits"] = nv.linear(x, router)
    y = check(nv, d, 2)
    assert not y[2].any()  # a padding token: no row, no contribution of any expert
    logits = nv.linear(y, table)
    r = nv.token_logprobs(logits, tokens, top_k=3, entropy=True)
    want = torch.log_softmax(y.double() @ table.double().t(), 1)
    live = tokens >= 0
    # the logits are rounded to 16 bits: each by 2^-9 of itself, and so is their log sum exp
    limit = 2 * (2.0 ** -9 + 2.0 ** -14) * logits.abs().amax(1).double() + 1e-4
    assert ((r.logprobs.double() - want[torch.arange(6), tokens.clamp_min(0)]).abs() <= limit)[live].all()
    op = torch.ops.nvfp4_b200.moe_layer(x, d["logits"], d["w13"], d["w2"], 2, "softmax", None, True, 1.0, x)
    assert torch.equal(op, y)


def test_example(nv, cuda_dev):
    """examples/moe_layer.py's decode step runs; its loss's gradients against 64 bits with the same
    choice of experts.  Some ten results on the way are rounded by at most 2^-8 of themselves, so
    a gradient is off by at most 10 2^-8 of its norm."""
    path = os.path.join(os.path.dirname(nv.__file__), "..", "examples", "moe_layer.py")
    spec = importlib.util.spec_from_file_location("example_moe_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    V, K, F, E, T, k = 96, 64, 32, 8, 24, 2
    g = gen(3)
    table, router = (torch.randn(r, K, device="cuda", generator=g).mul(K ** -0.5).bfloat16() for r in (V, E))
    w13 = (torch.randn(E * 2 * F, K, device="cuda", generator=g) * K ** -0.5).bfloat16()
    w2 = (torch.randn(E * K, F, device="cuda", generator=g) * F ** -0.5).bfloat16()
    tokens, targets = (torch.randint(0, V, (T,), device="cuda", generator=g) for _ in range(2))
    targets[3] = -100
    r = example.decode(tokens[:5], table, router, w13, w2, k)
    assert r.top_tokens.shape == (5, 5) and torch.isfinite(r.entropy).all()
    params = [t.requires_grad_() for t in (table, router, w13, w2)]
    got = torch.autograd.grad(example.loss(tokens, targets, *params, k), params)

    x = nv.embedding(tokens, table.detach(), K ** 0.5)
    experts = nv.moe_route(nv.linear(x, router.detach()), k).experts.long()
    p64 = [t.detach().double().requires_grad_() for t in params]
    t64, r64, a64, b64 = p64
    x = t64[tokens] * K ** 0.5
    logits = x @ r64.t()
    weights = torch.softmax(logits.gather(1, experts), 1)  # renormalised over the chosen ones
    h = R.act64(torch.einsum("tk,tjfk->tjf", x, a64.view(E, 2 * F, K)[experts]).reshape(T * k, 2 * F), "swiglu")
    y = x + (weights[:, :, None] * torch.einsum("tjf,tjkf->tjk", h.view(T, k, F), b64.view(E, K, F)[experts])).sum(1)
    logp = torch.log_softmax(y @ t64.t(), 1).gather(1, targets.clamp_min(0)[:, None])[:, 0]
    want = torch.autograd.grad(-(logp * (targets >= 0)).sum() / T, p64)
    for name, a, b in zip(("table", "router", "w13", "w2"), got, want):
        assert (a.double() - b).norm() <= 10 * 2.0 ** -8 * b.norm(), name
