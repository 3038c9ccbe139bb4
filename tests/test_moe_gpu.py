"""The router and the movement of rows on the GPU against plain 64-bit forms: masks that
leave a token nothing, ties, every expert count and top-k, gradients, and a whole layer."""
import math

import pytest
import torch

import ref16 as R

pytestmark = pytest.mark.gpu


def logits_of(T, E, dtype, seed, masked=0.0, ties=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * 2
    if ties:
        x = x.round()
    if masked:
        x[torch.rand(T, E, generator=g) < masked] = -math.inf
        x[::7] = -math.inf
    return x.to(dtype).cuda()


def check_route(nv, logits, k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    r = nv.moe_route(logits, k, scoring=scoring, bias=bias, renormalize=renormalize, scale=scale)
    w, e, rows, offs = R.route64(logits, k, scoring, bias, renormalize, scale)
    assert torch.equal(r.experts.cpu(), e)
    assert torch.equal(r.m_offsets.cpu(), offs)
    assert torch.equal(r.rows.cpu(), rows)
    # a score is a few fp32 operations (each 2^-23 relative) and a sum over at most 256 of them
    assert torch.allclose(r.weights.cpu().double(), w, rtol=1e-5, atol=1e-30)
    return r


@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (8, 2), (31, 3), (32, 32), (33, 1), (60, 4), (64, 6), (100, 8),
                                 (128, 5), (160, 6), (255, 8), (256, 32)])
@pytest.mark.parametrize("T", [1, 3, 33, 128, 129, 300])
def test_route_sizes(nv, cuda_dev, T, E, k):
    check_route(nv, logits_of(T, E, torch.bfloat16, T + E), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scoring,bias,renorm", [("softmax", False, True), ("softmax", False, False),
                                                 ("sigmoid", False, True), ("sigmoid", True, True),
                                                 ("sigmoid", True, False)])
def test_route_forms(nv, cuda_dev, dtype, scoring, bias, renorm):
    for masked, ties in ((0.0, False), (0.3, False), (0.1, True), (0.9, False)):
        l = logits_of(150, 40, dtype, 5, masked, ties)
        b = torch.randn(40, generator=torch.Generator().manual_seed(1)).cuda() * 0.1 if bias else None
        check_route(nv, l, 4, scoring, b, renorm, 2.5)


def test_route_masks(nv, cuda_dev):
    """Lowest finite values, -inf, NaN, signed zeros, and rows that nothing is left of."""
    low = torch.finfo(torch.float32).min
    l = torch.zeros(9, 6, device="cuda")
    l[0] = -math.inf                      # nothing left
    l[1] = low                            # all at the lowest value: equal, the first ones
    l[2, 1:] = -math.inf                  # one expert left
    l[3, ::2] = math.nan                  # NaN counts as masked
    l[4, 3] = -0.0                        # -0 and 0 are equal: the first ones
    l[4, 0] = -1.0
    l[5, 2] = low
    l[5, :2] = -math.inf
    l[6] = math.nan
    l[7] = torch.tensor([1e30, 2e30, -1e30, 0.0, 3e38, -3e38], device="cuda")
    r = nv.moe_route(l, 3)
    w, e, rows, offs = R.route64(torch.where(l.isnan(), torch.full_like(l, -math.inf), l), 3, "softmax", None, True, 1.0)
    assert torch.equal(r.experts.cpu(), e) and torch.equal(r.rows.cpu(), rows) and torch.equal(r.m_offsets.cpu(), offs)
    assert torch.allclose(r.weights.cpu().double(), w, rtol=1e-5)
    assert (r.experts[0] == -1).all() and (r.weights[0] == 0).all() and (r.rows[0] == -1).all()
    r = nv.moe_route(l[:7], 3, scoring="sigmoid")
    assert torch.isfinite(r.weights).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("E,k", [(33, 4), (64, 8), (100, 6), (128, 8), (200, 8), (256, 1), (256, 8), (256, 32)])
def test_biased_choice(nv, cuda_dev, E, k, dtype):
    """Sigmoid scores with a bias at two, four and eight experts a lane: exact ties (more
    experts at the top than candidates are kept), scores one rounding apart, and masks."""
    T = 40
    g = torch.Generator().manual_seed(E + k)
    l = torch.randn(T, E, generator=g) * 2
    l[:8] = l[:8].round()                                # tied scores
    l[8:12] = 0.5                                        # all tied
    l[12:16] = 1.0 + torch.randint(0, 4, (4, E), generator=g) * 2.0 ** -22  # a few fp32 roundings apart
    l[16:20] = 30.0 + torch.rand(4, E, generator=g)      # scores that round to 1
    l[20:24] = -60.0 - torch.rand(4, E, generator=g)     # scores far below the bias's rounding
    l[24:28][:, ::2] = -math.inf
    l[28] = -math.inf
    l[29, 1:] = -math.inf
    l = l.to(dtype).cuda()
    bias = torch.randn(E, generator=g) * 0.05
    for b in (torch.zeros(E), bias, bias.bfloat16().float(), torch.full((E,), 0.25), bias * 1e4):
        for renorm in (True, False):
            check_route(nv, l, k, "sigmoid", b.cuda(), renorm)


@pytest.mark.parametrize("T,E,k", [(0, 8, 2), (5000, 256, 8), (40_000, 16, 3)])
def test_route_many_tokens(nv, cuda_dev, T, E, k):
    """Every row is used once, in order of expert and token (several chunks of tokens)."""
    l = logits_of(T, E, torch.bfloat16, 3, 0.05, ties=True)
    r = nv.moe_route(l, k)
    flat, rows = r.experts.flatten(), r.rows.flatten()
    live = flat >= 0
    n = int(live.sum())
    assert int(r.m_offsets[-1]) == n and int(r.m_offsets[0]) == 0
    assert torch.equal(torch.sort(rows[live]).values, torch.arange(n, device="cuda", dtype=torch.int32))
    assert (rows[~live] == -1).all()
    order = torch.sort(torch.where(live, flat, E), stable=True).indices[:n]
    assert torch.equal(rows[order], torch.arange(n, device="cuda", dtype=torch.int32))
    assert torch.equal(torch.diff(r.m_offsets), torch.bincount(flat[live].long(), minlength=E).int())
    top = torch.sort(l.float(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(torch.where(r.experts >= 0, r.experts, 0),
                       torch.where(r.experts >= 0, top, 0).int())
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(r, nv.moe_route(l, k)))


def test_scores_round_as_the_formula(nv, cuda_dev):
    """The score that a bias is added to has the plain fp32 formula's bits for every bf16
    value, so the ranking of near-ties is the formula's."""
    v = torch.arange(-(1 << 15), 1 << 15, device="cuda").to(torch.int16).view(torch.bfloat16)
    v = v[v.float().isfinite()]
    r = nv.moe_route(v[:, None].contiguous(), 1, scoring="sigmoid", renormalize=False)
    assert torch.equal(r.weights[:, 0], 1 / (1 + torch.exp(-v.float())))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T,E,k,masked", [(1, 2, 1, 0.0), (20, 8, 2, 0.0), (37, 33, 5, 0.3), (9, 256, 32, 0.9),
                                          (70, 100, 8, 0.1)])
def test_route_backward(nv, cuda_dev, scoring, renorm, T, E, k, masked):
    """Against autograd in 64 bits on the same choice, and against differences of the
    weights; fp32 logits: the gradient's error is a few fp32 roundings of its largest term."""
    l = logits_of(T, E, torch.float32, 7, masked)
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(2)).cuda()
    r = nv.moe_route(l, k, scoring=scoring, renormalize=renorm, scale=1.5)
    got = nv.moe_route_backward(dw, l, r, scoring=scoring, renormalize=renorm, scale=1.5)
    x = l.double().requires_grad_()

    def weights(x):
        dead = l == -math.inf
        if scoring == "sigmoid":
            s = torch.sigmoid(x)
        else:
            s = torch.softmax(x.masked_fill(dead.all(1, keepdim=True), 0.0), 1)
        p = torch.gather(s, 1, r.experts.long().clamp_min(0)) * (r.experts >= 0)
        if renorm:
            t = p.sum(1, keepdim=True)
            p = p / torch.where(t > 0, t, torch.ones_like(t))
        return 1.5 * p

    ref = torch.autograd.grad((weights(x) * dw.double()).sum(), x)[0].nan_to_num()
    bound = 1e-5 * dw.abs().sum(1, keepdim=True).double() * 1.5
    assert ((got.double() - ref).abs() <= bound).all()
    d = torch.randn(T, E, generator=torch.Generator().manual_seed(3)).cuda().double()
    h = 1e-5
    diff = (((weights(l.double() + h * d) - weights(l.double() - h * d)) / (2 * h)) * dw.double()).sum(1)
    assert ((got.double() * d).sum(1) - diff).abs().max() <= 1e-4 * dw.abs().sum(1).max() * d.abs().max()


def routing_of(nv, T, E, k, masked, seed=1):
    return nv.moe_route(logits_of(T, E, torch.float32, seed, masked), k)


MOVES = [(1, 2, 1, 8, 0.0), (5, 4, 2, 24, 0.0), (32, 8, 2, 4096, 0.0), (33, 16, 5, 256, 0.3), (130, 64, 8, 264, 0.1),
         (300, 128, 32, 72, 0.2), (64, 8, 3, 8200, 0.5), (1000, 8, 1, 520, 0.0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,K,masked", MOVES)
def test_move(nv, cuda_dev, T, E, k, K, masked, dtype):
    r = routing_of(nv, T, E, k, masked)
    gen = torch.Generator().manual_seed(4)
    x, res, dy = (torch.randn(T, K, generator=gen).to(dtype).cuda() for _ in range(3))
    er, dr = (torch.randn(T * k, K, generator=gen).to(dtype).cuda() for _ in range(2))
    n = int(r.m_offsets[-1])
    er[n:] = math.nan  # rows that no choice owns are never read
    live, rows, w = r.rows >= 0, r.rows.long(), r.weights.double()
    token = torch.arange(T, device="cuda")[:, None].expand(T, k)

    xs = nv.moe_dispatch(x, r)
    ref = torch.zeros_like(er)
    ref[rows[live]] = x[token[live]]
    assert torch.equal(xs, ref)

    picked = torch.where(live[..., None], er[rows.clamp_min(0)].double(), 0.0)
    for residual in (None, res):
        y = nv.moe_combine(er, r, residual=residual)
        ref = (picked * w[..., None]).sum(1) + (0 if residual is None else res.double())
        # k products and sums in fp32
        bound = (k + 2) * 2.0 ** -23 * ((picked * w[..., None]).abs().sum(1) + res.double().abs())
        R.assert_close(y, ref, bound, "combine")

    dx = nv.moe_dispatch_backward(dr, r)
    pd = torch.where(live[..., None], dr[rows.clamp_min(0)].double(), 0.0)
    R.assert_close(dx, pd.sum(1), (k + 1) * 2.0 ** -23 * pd.abs().sum(1), "dispatch backward")

    drows, dw = nv.moe_combine_backward(dy, er, r)
    ref = torch.zeros(T * k, K, dtype=torch.float64, device="cuda")
    ref[rows[live]] = (dy.double()[:, None] * w[..., None])[live]
    R.assert_close(drows, ref, 2.0 ** -23 * ref.abs(), "drows")
    ref = (picked * dy.double()[:, None]).sum(2)
    bound = (K / 64 + 16) * 2.0 ** -23 * (picked * dy.double()[:, None]).abs().sum(2)
    assert ((dw.double() - ref).abs() <= bound).all()
    assert (dw[~live] == 0).all()


def test_layer_forward_and_backward(nv, cuda_dev):
    """Router, dispatch, SwiGLU experts, down projection, combine with residual, and back,
    against autograd in 64 bits.  Each stage rounds to bf16, which the 64-bit pass does not:
    a relative error of a few u = 2^-8 in the norm."""
    T, E, k, K, F, dt = 150, 8, 2, 128, 96, torch.bfloat16
    gen = torch.Generator().manual_seed(9)

    def rnd(*s, scale=1.0):
        return (torch.randn(*s, generator=gen) * scale).to(dt).cuda()

    x, wr = rnd(T, K), rnd(E, K, scale=K ** -0.5)
    w1, w2 = rnd(E * 2 * F, K, scale=K ** -0.5), rnd(E * K, F, scale=F ** -0.5)
    dy = rnd(T, K)
    logits = nv.linear(x, wr)
    r = nv.moe_route(logits, k)
    xs = nv.moe_dispatch(x, r)
    h, z = nv.linear_grouped(xs, w1, r.m_offsets, activation="swiglu", return_preact=True)
    ys = nv.linear_grouped(h, w2, r.m_offsets)
    y = nv.moe_combine(ys, r, residual=x)
    dys, dwt = nv.moe_combine_backward(dy, ys, r)
    dh, dw2, _ = nv.linear_grouped_backward(dys, h, w2, r.m_offsets)
    dxs, dw1, _ = nv.linear_grouped_backward(dh, xs, w1, r.m_offsets, preact=z, activation="swiglu")
    dl = nv.moe_route_backward(dwt, logits, r)
    dxr, dwr, _ = nv.linear_backward(dl, x, wr)
    dx = dy.double() + nv.moe_dispatch_backward(dxs, r).double() + dxr.double()
    nv.device_status()

    p = [t.double().requires_grad_() for t in (x, wr, w1, w2)]
    lg = p[0] @ p[1].t()
    wt = torch.softmax(torch.gather(lg, 1, r.experts.long()), 1)
    out = p[0]
    for j in range(k):
        e = r.experts[:, j].long()
        a = p[2].view(E, 2 * F, K)[e]
        hh = R.act64(torch.bmm(a, p[0][:, :, None])[..., 0], "swiglu")
        out = out + wt[:, j:j + 1] * torch.bmm(p[3].view(E, K, F)[e], hh[:, :, None])[..., 0]
    grads = torch.autograd.grad((out * dy.double()).sum(), p)
    for got, ref, n in ((y, out, "y"), (dx, grads[0], "dx"), (dwr, grads[1], "dwr"), (dw1, grads[2], "dw1"),
                        (dw2, grads[3], "dw2")):
        rel = ((got.double() - ref).norm() / ref.norm()).item()
        assert rel <= 4 * R.U[dt], f"{n}: {rel}"


def test_nvfp4_experts_take_the_routing(nv, cuda_dev):
    """The same routing drives the NVFP4 experts: quantize_grouped and gemm_grouped on the
    dispatched rows and m_offsets; against the 16-bit experts with the dequantized operands'
    error (e2m1 with one scale per 16: a few percent in the norm)."""
    T, E, k, K, N = 200, 4, 2, 256, 128
    gen = torch.Generator().manual_seed(11)
    x = torch.randn(T, K, generator=gen).bfloat16().cuda()
    w = (torch.randn(E * N, K, generator=gen) * K ** -0.5).bfloat16().cuda()
    r = nv.moe_route(torch.randn(T, E, generator=gen).cuda(), k)
    xs = nv.moe_dispatch(x, r)
    _, gx = nv.global_scale(xs)
    _, gw = nv.global_scale(w)
    q, sf = nv.quantize_grouped(xs, gx, r.m_offsets)
    wq, wsf = nv.quantize(w, gw)
    y4 = nv.moe_combine(nv.gemm_grouped(q, sf, wq, wsf, (gx * gw).expand(E).contiguous(), r.m_offsets), r)
    y16 = nv.moe_combine(nv.linear_grouped(xs, w, r.m_offsets), r)
    nv.device_status()
    assert ((y4.double() - y16.double()).norm() / y16.double().norm()).item() < 0.25


def test_refusals(nv, cuda_dev):
    l = logits_of(8, 16, torch.float32, 1)
    x = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    r = nv.moe_route(l, 2)
    for bad in (lambda: nv.moe_route(l.double(), 2), lambda: nv.moe_route(l[:, ::2], 2), lambda: nv.moe_route(l[0], 2),
                lambda: nv.moe_route(l, 2, scoring="tanh"), lambda: nv.moe_route(l, 2, bias=l[0]),
                lambda: nv.moe_route(l, 2, scoring="sigmoid", bias=l[0].bfloat16()),
                lambda: nv.moe_dispatch(x[:4], r), lambda: nv.moe_dispatch(x[:, :60].contiguous(), r),
                lambda: nv.moe_dispatch(x.float(), r), lambda: nv.moe_combine(x, r),
                lambda: nv.moe_dispatch(x, (r.weights, r.experts)),
                lambda: nv.moe_combine_backward(x[:4], torch.zeros(16, 64, dtype=torch.bfloat16, device="cuda"), r),
                lambda: nv.moe_route_backward(r.weights[:4], l, r)):
        with pytest.raises(ValueError):
            bad()
    for k in (0, 17):
        with pytest.raises(nv.NVFP4Error):
            nv.moe_route(l, k)
    with pytest.raises(nv.NVFP4Error):
        nv.moe_route(torch.zeros(4, 300, device="cuda"), 2)


def test_route_from_two_threads(nv, cuda_dev):
    """Two threads route numbers of tokens that need different amounts of shared memory (more
    than 262144 tokens of 256 experts), at the same time: neither call fails, and every row
    is numbered as by the other calls of the same logits."""
    import threading
    E, k, errors = 256, 2, []
    logits = [torch.randn(T, E, device="cuda", generator=torch.Generator("cuda").manual_seed(T)).bfloat16()
              for T in (1 << 20, 300_000)]
    first = [nv.moe_route(l, k) for l in logits]
    for l, r in zip(logits, first):
        flat = r.experts.flatten().long()
        order = torch.sort(flat, stable=True).indices
        assert torch.equal(r.rows.flatten()[order], torch.arange(len(flat), device="cuda", dtype=torch.int32))
        assert torch.equal(torch.diff(r.m_offsets), torch.bincount(flat, minlength=E).int())
        assert torch.equal(r.experts[:, 0].long(), l.float().max(1).indices)
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    r = nv.moe_route(logits[i], k)
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(r, first[i]))
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
