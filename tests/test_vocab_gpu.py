"""GPU: embedding and token log probabilities, with their gradients, against plain 64-bit forms."""
import math

import pytest
import torch

import ref16 as R
import ref_vocab as V

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tokens_of(T, rows, seed, dtype=torch.int64, common=0.3, padded=0.1):
    """Uniform tokens, a share of them the same one, some outside the table."""
    g = gen(seed)
    t = torch.randint(0, rows, (T,), device="cuda", generator=g)
    t[torch.rand(T, device="cuda", generator=g) < common] = rows // 2
    out = torch.rand(T, device="cuda", generator=g) < padded
    t[out] = torch.where(torch.rand(int(out.sum()), device="cuda", generator=g) < 0.5, -1, rows)
    return t.to(dtype)


# ------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,rows,K", [(1, 1, 8), (1, 50, 4096), (7, 300, 264), (16, 1000, 8200), (333, 40, 72),
                                      (4097, 129, 2048)])
@pytest.mark.parametrize("scale", [1.0, 45.254833995939045, -0.3])
def test_embedding(nv, cuda_dev, dtype, T, rows, K, scale):
    table = torch.randn(rows, K, device="cuda", generator=gen(T)).to(dtype)
    for index in (torch.int64, torch.int32):
        t = tokens_of(T, rows, T + rows, index)
        y = nv.embedding(t, table, scale)
        ref = V.embedding64(t, table, scale)
        if scale == 1.0:
            assert torch.equal(y.double(), ref)
        R.assert_close(y, ref, 2.0 ** -23 * ref.abs())  # the scale's own rounding, the product's


def test_embedding_shapes_and_rows(nv, cuda_dev):
    wide = torch.randn(50, 128, device="cuda", generator=gen(1)).bfloat16()
    table = wide[:, 32:96]  # rows of wider ones
    t = torch.tensor([[[1, 49], [0, 50], [-1, 2 ** 40]]], device="cuda")
    y = nv.embedding(t, table)
    assert y.shape == (1, 3, 2, 64) and torch.equal(y.double(), V.embedding64(t, table, 1.0))
    assert not y[0, 1, 1].any() and not y[0, 2].any()
    assert nv.embedding(t[:0], table).shape == (0, 3, 2, 64)
    assert nv.embedding(t[0, 0, 0], table).shape == (64,)
    bits = torch.tensor([[0x7fc1, 0x7f80, 0x8000, 0x0001] * 2], dtype=torch.int32).to(torch.int16).view(torch.bfloat16).cuda()
    out = nv.embedding(torch.zeros(3, dtype=torch.int32, device="cuda"), bits)
    assert torch.equal(out.view(torch.int16), bits.view(torch.int16).expand(3, 8))  # NaN, inf, -0, subnormal


def check_embedding_backward(nv, dy, t, rows, scale=1.0):
    d = nv.embedding_backward(dy, t, rows, scale)
    ref, bound = V.embedding_backward64(dy, t, rows, scale)
    R.assert_close(d, ref, bound + 2.0 ** -23 * ref.abs())
    assert not d[torch.bincount(t.reshape(-1).clamp(-1, rows).long() + 1, minlength=rows + 2)[1:-1] == 0].any()
    return d


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,rows,K", [(1, 1, 8), (1, 70, 4096), (31, 5, 64), (32, 5, 64), (33, 5, 72), (64, 1, 2056),
                                      (65, 1000, 128), (1000, 63, 264), (4096, 64, 40), (4096, 5000, 256),
                                      (7, 300, 8200), (900, 40, 1032), (1024, 3000, 520), (1025, 9, 8), (2047, 700, 2056),
                                      (2048, 30, 16), (2049, 30, 64), (129, 2000, 4104)])
def test_embedding_backward_small(nv, cuda_dev, dtype, T, rows, K):
    dy = torch.randn(T, K, device="cuda", generator=gen(T)).to(dtype)
    for seed, (common, padded) in enumerate([(0.0, 0.0), (0.5, 0.2), (1.0, 0.0), (0.0, 1.0)]):
        index = torch.int32 if seed % 2 else torch.int64
        check_embedding_backward(nv, dy, tokens_of(T, rows, seed, index, common, padded), rows, 0.5 + seed)


@pytest.mark.parametrize("T,rows,K", [(4097, 3, 64), (5000, 511, 64), (8191, 512, 24), (40000, 100000, 128),
                                      (33000, 270000, 64), (140001, 7, 32), (270000, 1 << 20, 8)])
def test_embedding_backward_radix(nv, cuda_dev, T, rows, K):
    """More tokens than one CTA sorts: one, two and three passes, odd digits, blocks of every
    length, more than one tile a chunk, runs over many blocks."""
    dy = torch.randn(T, K, device="cuda", generator=gen(T)).bfloat16()
    for seed, common in enumerate((0.0, 0.3, 1.0)):
        check_embedding_backward(nv, dy, tokens_of(T, rows, seed, common=common), rows)


def test_embedding_backward_forms(nv, cuda_dev):
    g = gen(3)
    wide = torch.randn(200, 256, device="cuda", generator=g).bfloat16()
    t = tokens_of(200, 30, 5)
    a = check_embedding_backward(nv, wide[:, 64:128], t, 30)  # rows of wider ones
    b = nv.embedding_backward(wide[:, 64:128].contiguous().view(4, 50, 64), t.view(4, 50), 30)
    assert torch.equal(a, b)
    # rows of ignored tokens are not read
    dy = wide[:, :64].clone()
    dy[(t < 0) | (t >= 30)] = math.nan
    assert torch.isfinite(nv.embedding_backward(dy, t, 30)).all()
    z = nv.embedding_backward(dy[:0], t[:0], 30)
    assert z.shape == (30, 64) and not z.any()
    with pytest.raises(ValueError):
        nv.embedding_backward(dy, t[:10], 30)
    with pytest.raises(ValueError):
        nv.embedding_backward(dy, t, 0)
    with pytest.raises(ValueError):
        nv.embedding(t.float(), dy)
    with pytest.raises(ValueError):
        nv.embedding(t, dy[:, :60])
    with pytest.raises(ValueError):
        nv.embedding(t, dy, math.nan)
    with pytest.raises(ValueError):
        nv.embedding(t, dy.float())


def test_embedding_backward_order(nv, cuda_dev):
    """The tokens' order alone decides the sum: the same bits every time, and rows whose sum
    depends on the order (1e4 + many small ones) come out as the formula of one order."""
    T = 9000
    t = torch.full((T,), 3, device="cuda")
    dy = torch.full((T, 64), 2.0 ** -12, device="cuda").bfloat16()
    dy[0] = 256.0
    a = nv.embedding_backward(dy, t, 5)
    for _ in range(3):
        assert torch.equal(a, nv.embedding_backward(dy, t, 5))
    check_embedding_backward(nv, dy, t, 5)


# ------------------------------------------------------------------------- log probabilities
def logits_of(T, W, dtype, seed, masked=0.0):
    g = gen(seed)
    x = torch.randn(T, W, device="cuda", generator=g) * 3
    if masked:
        x[torch.rand(T, W, device="cuda", generator=g) < masked] = -math.inf
    return x.to(dtype)


def targets_of(T, vocab, seed, dtype=torch.int64):
    g = gen(seed)
    t = torch.randint(0, vocab, (T,), device="cuda", generator=g)
    t[torch.rand(T, device="cuda", generator=g) < 0.2] = -100
    if T > 2:
        t[1] = vocab  # the first outside
    return t.to(dtype)


def check_logprobs(nv, x, t, vocab=None, k=0, temperature=1.0, entropy=True, grad=True, out=None):
    n = x.shape[1] if vocab is None else vocab
    r = nv.token_logprobs(x, t, vocab, k, temperature, entropy)
    ref = V.Logprobs(x, t, n, k, temperature)
    V.assert_near(r.logprobs, ref.logprobs, ref.logprobs_bound, "logprobs")
    V.assert_near(r.lse, ref.lse, ref.lse_bound, "lse")
    if entropy:
        V.assert_near(r.entropy, ref.entropy, ref.entropy_bound, "entropy")
    else:
        assert r.entropy is None
    if k:
        assert torch.equal(r.top_tokens.long(), ref.top_tokens)
        size = torch.where(ref.top_logprobs.isinf(), torch.zeros_like(ref.top_logprobs), ref.top_logprobs.abs())
        V.assert_near(r.top_logprobs, ref.top_logprobs, ref.logprobs_bound[:, None] + 2.0 ** -21 * size, "top")
    else:
        assert r.top_tokens is None and r.top_logprobs is None
    if grad:
        g = gen(9)
        dl, dh = torch.randn(len(t), device="cuda", generator=g), torch.randn(len(t), device="cuda", generator=g)
        want, bound = ref.grad(dl, dh if entropy else None, x.shape[1])
        d = nv.token_logprobs_backward(dl, x, t, r, dh if entropy else None, vocab, temperature, out)
        V.assert_grad(d, want, bound, "dlogits")
    return r


@pytest.mark.parametrize("dtype", DT + [torch.float32])
@pytest.mark.parametrize("T,vocab,W", [(1, 1, 1), (3, 7, 7), (2, 8, 16), (5, 1000, 1003), (33, 4099, 4104),
                                       (149, 511, 512), (400, 9001, 9001), (1, 50257, 50264), (9, 131072, 131072),
                                       (2, 262143, 262143)])
def test_logprobs(nv, cuda_dev, dtype, T, vocab, W):
    x = logits_of(T, W, dtype, T + vocab)
    for i, (k, entropy, temperature) in enumerate([(0, False, 1.0), (5, True, 0.7), (32, False, 1.0), (0, True, 2.5),
                                                   (1, True, 1.0), (20, True, 1.0)]):
        t = targets_of(T, vocab, i, torch.int32 if i % 2 else torch.int64)
        check_logprobs(nv, x, t, vocab, k, temperature, entropy)


@pytest.mark.parametrize("dtype", DT + [torch.float32])
def test_logprobs_rows_of_any_alignment(nv, cuda_dev, dtype):
    wide = logits_of(70, 5011, dtype, 4)
    t = targets_of(70, 3000, 1)
    for first in (0, 1, 3, 8, 9):
        x = wide[:, first:first + 4001]
        check_logprobs(nv, x, t, 3001, 7)
        check_logprobs(nv, x, t, 3001, 0, out=torch.empty_like(wide)[:, first:first + 4001])
        check_logprobs(nv, x, t, 3001, 0, out=torch.empty_like(wide)[:, first + 1:first + 4002])
        check_logprobs(nv, x[5:6], t[5:6], None, 3)


def test_logprobs_gradient_in_place(nv, cuda_dev):
    for x in (logits_of(50, 1001, torch.bfloat16, 1), logits_of(50, 1100, torch.float32, 2)[:, 3:1004]):
        t = targets_of(50, 1001, 1)
        g = torch.randn(50, device="cuda", generator=gen(1))
        r = nv.token_logprobs(x, t, entropy=True)
        want = nv.token_logprobs_backward(g, x, t, r, g)
        got = nv.token_logprobs_backward(g, x, t, r, g, out=x)
        assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("dtype", DT + [torch.float32])
@pytest.mark.parametrize("vocab", [40, 3000, 140000])
def test_logprobs_masks(nv, cuda_dev, dtype, vocab):
    """Masked tokens (-inf, NaN), a masked target, the type's lowest value, nothing left, fewer
    tokens left than alternatives."""
    x = logits_of(12, vocab, dtype, 5, masked=0.5)
    t = targets_of(12, vocab, 3)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = low
    x[3] = -math.inf
    x[3, 7] = 1.5
    x[3, vocab - 1] = low
    x[4, ::3] = math.nan
    x[5] = low
    x[5, 9] = 3.0
    t[0], t[1], t[2], t[3], t[4], t[5] = 1, 2, 3, 8, 6, 9
    for k in (0, 5, 32):
        r = check_logprobs(nv, x, t, None, k)
        assert r.logprobs[0] == r.logprobs[1] == -math.inf and r.entropy[0] == r.entropy[1] == 0
        if k:
            assert (r.top_tokens[:2] == -1).all() and r.top_tokens[3, 0] == 7 and r.top_tokens[3, 1] == vocab - 1
            assert r.top_tokens[3, 2] == -1
    # no gradient where there is no probability, even for a masked target
    g = torch.ones(12, device="cuda")
    d = nv.token_logprobs_backward(g, x, t, r, g)
    assert not d[~(x > -math.inf)].any() and torch.isfinite(d).all()


def test_logprobs_infinite_logit(nv, cuda_dev):
    x = logits_of(3, 500, torch.float32, 1)
    x[1, 100] = math.inf
    t = torch.tensor([4, 5, 6], device="cuda")
    r = nv.token_logprobs(x, t, top_k=2, entropy=True)
    assert r.logprobs[1].isnan() and r.entropy[1].isnan() and r.lse[1].isnan() and r.top_tokens[1, 0] == 100
    d = nv.token_logprobs_backward(torch.ones(3, device="cuda"), x, t, r)
    assert d[1].isnan().any() and torch.isfinite(d[::2]).all() and torch.isfinite(r.logprobs[::2]).all()


@pytest.mark.parametrize("T", [2, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_ties(nv, cuda_dev, dtype, T):
    """Equal logits: whole rows of them, a few values only, both zeros, rows in order."""
    n = 20000
    x = torch.zeros(T, n, device="cuda")
    x[0] = 2.5
    x[1] = torch.randint(0, 3, (n,), device="cuda", generator=gen(1)).float()
    if T > 2:
        x[2] = torch.arange(n, device="cuda") / n           # ascending
        x[3] = -torch.arange(n, device="cuda") / n          # descending
        x[4, ::2] = -0.0                                    # zeros of both signs
        x[5, 19000:] = 1.0                                  # a run at the end
        x[6, 5::512] = torch.arange(len(x[6, 5::512]), device="cuda").float()
        x[7, :4096] = torch.arange(4096, device="cuda").float()  # all candidates with one thread's column
        x[8, 19999] = 3.0
        x[9] = -math.inf
        x[9, 600:700] = 1.0
    x = x.to(dtype)
    t = targets_of(T, n, 1)
    for k in (1, 20, 32):
        check_logprobs(nv, x, t, None, k, grad=False)


@pytest.mark.parametrize("dtype", DT + [torch.float32])
@pytest.mark.parametrize("T,vocab,W", [(600, 1, 1), (641, 7, 7), (600, 40, 40), (700, 1000, 1003), (650, 2040, 2056),
                                       (1300, 4001, 4001), (2500, 8100, 8104)])
def test_logprobs_many_short_rows(nv, cuda_dev, dtype, T, vocab, W):
    """Rows that a warp takes each, and gradients of several rows a CTA."""
    x = logits_of(T, W, dtype, vocab)
    for k, entropy, temperature in ((0, False, 1.0), (8, True, 0.7), (32, True, 1.0)):
        check_logprobs(nv, x, targets_of(T, vocab, k), vocab, k, temperature, entropy)


@pytest.mark.parametrize("dtype", DT + [torch.float32])
@pytest.mark.parametrize("n", [9, 300, 3001])
def test_logprobs_many_short_rows_forms(nv, cuda_dev, dtype, n):
    """The same with masks, ties, rows of any alignment, maxima that move at every step."""
    T = 1000
    low = torch.finfo(dtype).min
    wide = logits_of(T, n + 20, dtype, 3, masked=0.4)
    for first in (0, 1, 5, 8):
        x = wide[:, first:first + n]
        x[0] = -math.inf
        x[1] = math.nan
        x[2] = low
        x[3] = -math.inf
        x[3, 7] = 1.5
        x[4, ::3] = math.nan
        x[5] = 2.5
        x[6] = torch.randint(0, 3, (n,), device="cuda", generator=gen(1)).to(dtype)
        x[7] = (torch.arange(n, device="cuda") / 8).to(dtype)
        x[8] = (-torch.arange(n, device="cuda") / 8).to(dtype)
        x[9] = torch.linspace(-3e4, 3e4, n).to(dtype)
        t = targets_of(T, n, first)
        t[0], t[3], t[4], t[9] = 2, 7, 3, n - 1
        for k in (0, 1, 8, 20, 32):
            r = check_logprobs(nv, x, t, None, k)
            assert r.logprobs[0] == -math.inf and r.entropy[0] == 0
        check_logprobs(nv, x, t, None, 0, out=torch.empty_like(wide)[:, first + 1:first + n + 1])
        d = nv.token_logprobs_backward(torch.ones(T, device="cuda"), x, t, r, torch.ones(T, device="cuda"))
        assert not d[~(x > -math.inf)].any() and torch.isfinite(d).all()
        own = x.clone()
        assert torch.equal(nv.token_logprobs_backward(torch.ones(T, device="cuda"), own, t, r,
                                                      torch.ones(T, device="cuda"), out=own), d)


def test_logprobs_far_values(nv, cuda_dev):
    """Probabilities that underflow, and maxima that move at every step."""
    n = 9000
    x = torch.zeros(4, n, device="cuda")
    x[0] = torch.linspace(-3e4, 3e4, n)
    x[1] = torch.linspace(3e4, -3e4, n)
    x[2, 50] = 1e30
    x[3] = -1e30
    x[3, 3] = -1e30 * (1 - 2 ** -10)
    t = torch.tensor([n - 1, 0, 50, 3], device="cuda")
    for temperature in (1.0, 0.1, 50.0):
        check_logprobs(nv, x, t, None, 4, temperature)


def test_logprobs_differences(nv, cuda_dev):
    """The gradient against central differences of the kernel's own results.  With a step s the
    differences are off by s^2 / 6 times the third derivative (below 8 here) and by the results'
    errors (below 4e-6) over s."""
    x = torch.randn(3, 40, device="cuda", generator=gen(1)) * 2
    t = torch.tensor([3, 17, 39], device="cuda")
    g, h = torch.tensor([1.0, -0.5, 0.3], device="cuda"), torch.tensor([0.2, 0.7, -1.0], device="cuda")
    r = nv.token_logprobs(x, t, entropy=True)
    d = nv.token_logprobs_backward(g, x, t, r, h)
    s = 2.0 ** -6

    def loss(v):
        q = nv.token_logprobs(v, t, entropy=True)
        return (q.logprobs * g + q.entropy * h).double()

    for i in range(40):
        up, down = x.clone(), x.clone()
        up[:, i] += s
        down[:, i] -= s
        diff = (loss(up) - loss(down)) / (2 * s)
        assert (diff - d[:, i]).abs().max() <= s * s / 6 * 8 + 4e-6 / s


def test_vocab_same_bits(nv, cuda_dev):
    x = logits_of(40, 30000, torch.bfloat16, 1)
    t = targets_of(40, 30000, 1)
    first = nv.token_logprobs(x, t, top_k=20, entropy=True)
    for _ in range(5):
        for a, b in zip(first, nv.token_logprobs(x, t, top_k=20, entropy=True)):
            assert torch.equal(a, b)


def test_vocab_refusals(nv, cuda_dev):
    x, t = logits_of(4, 64, torch.float32, 1), targets_of(4, 64, 1)
    r = nv.token_logprobs(x, t)
    g = torch.ones(4, device="cuda")
    for call in (lambda: nv.token_logprobs(x.double(), t), lambda: nv.token_logprobs(x[0], t),
                 lambda: nv.token_logprobs(x.t(), t), lambda: nv.token_logprobs(x, t[:3]),
                 lambda: nv.token_logprobs(x, t.float()), lambda: nv.token_logprobs(x, t.cpu()),
                 lambda: nv.token_logprobs(x, t, vocab=65), lambda: nv.token_logprobs(x, t, vocab=0),
                 lambda: nv.token_logprobs(x, t, top_k=33), lambda: nv.token_logprobs(x, t, top_k=-1),
                 lambda: nv.token_logprobs(x, t, temperature=0.0),
                 lambda: nv.token_logprobs(x, t, temperature=math.nan),
                 lambda: nv.token_logprobs(x[:1].expand(4, 64), t),
                 lambda: nv.token_logprobs_backward(g[:3], x, t, r),
                 lambda: nv.token_logprobs_backward(g, x, t, r, g),
                 lambda: nv.token_logprobs_backward(g, x, t, r, out=x[:, :32]),
                 lambda: nv.token_logprobs_backward(g, x, t, r, out=x.bfloat16())):
        with pytest.raises(ValueError):
            call()
    both = torch.empty(8, 64, device="cuda")
    with pytest.raises(ValueError):  # overlaps the logits, but is not them
        nv.token_logprobs_backward(g, both[:4], t, r, out=both[1:5])
    empty = nv.token_logprobs(x[:0], t[:0], top_k=3, entropy=True)
    assert empty.top_tokens.shape == (0, 3) and empty.entropy.shape == (0,)
    assert nv.token_logprobs_backward(g[:0], x[:0], t[:0], empty).shape == (0, 64)


@pytest.mark.parametrize("seed", [0, 1])
def test_vocab_streams_and_graphs(nv, cuda_dev, seed):
    """On a side stream, and captured: replays follow inputs changed in place."""
    x, t = logits_of(20, 40000, torch.bfloat16, seed), targets_of(20, 40000, seed)
    table = torch.randn(40000, 64, device="cuda", generator=gen(seed)).bfloat16()
    tokens, dy = tokens_of(6000, 40000, seed), torch.randn(6000, 64, device="cuda", generator=gen(seed)).bfloat16()
    g = torch.randn(20, device="cuda", generator=gen(seed))

    def calls():
        r = nv.token_logprobs(x, t, top_k=8, entropy=True)
        return [*r, nv.token_logprobs_backward(g, x, t, r, g), nv.embedding(tokens, table, 2.0),
                nv.embedding_backward(dy, tokens, 40000, 2.0)]

    want = calls()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = calls()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls()
    for _ in range(2):
        x.copy_(logits_of(20, 40000, torch.bfloat16, seed + 50))
        tokens.copy_(tokens_of(6000, 40000, seed + 51))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, calls()))
        seed += 1


def test_vocab_autograd(nv, cuda_dev):
    """The differentiable operators: gradients of a loss through both, and of each alone."""
    ops = torch.ops.nvfp4_b200
    g = gen(2)
    table = (torch.randn(300, 64, device="cuda", generator=g) * 0.3).bfloat16().requires_grad_()
    tokens, targets = tokens_of(50, 300, 1), targets_of(50, 300, 2)
    x = ops.embedding(tokens, table, 3.0)
    logits = ops.linear_preact(x, table.detach()[:304 // 8 * 8 - 8])[0]  # 296 tokens
    logp, ent, top, tok, lse = ops.token_logprobs(logits, targets, 290, 4, 0.8, True)
    assert not top.requires_grad and not lse.requires_grad
    a, b = torch.randn(50, device="cuda", generator=g), torch.randn(50, device="cuda", generator=g)
    (logp * a + ent * b).sum().backward()
    r = nv.token_logprobs(logits.detach(), targets, 290, 4, 0.8, True)
    assert torch.equal(r.logprobs, logp) and torch.equal(r.top_tokens, tok)
    dl = nv.token_logprobs_backward(a, logits.detach(), targets, r, b, 290, 0.8)
    dx, _, _ = nv.linear_backward(dl, x.detach(), table.detach()[:296], weight_grad=False)
    assert torch.equal(table.grad, nv.embedding_backward(dx, tokens, 300, 3.0))
    # one result alone; no gradient through the alternatives
    leaf = logits.detach().requires_grad_()
    for entropy in (True, False):
        logp, ent, *_ = ops.token_logprobs(leaf, targets, None, 0, 1.0, entropy)
        d, = torch.autograd.grad(logp.sum(), leaf)
        r = nv.token_logprobs(leaf.detach(), targets, entropy=entropy)
        assert torch.equal(d, nv.token_logprobs_backward(torch.ones(50, device="cuda"), leaf.detach(), targets, r))
    logp, ent, *_ = ops.token_logprobs(leaf, targets, None, 0, 1.0, True)
    d, = torch.autograd.grad(ent.sum(), leaf)
    r = nv.token_logprobs(leaf.detach(), targets, entropy=True)
    one = torch.ones(50, device="cuda")
    assert torch.equal(d, nv.token_logprobs_backward(one * 0, leaf.detach(), targets, r, one))


def test_embedding_gradient_captured_beside_an_eager_graph(nv, cuda_dev):
    """A backward pass captured while an eager graph of the same leaves lives."""
    ops = torch.ops.nvfp4_b200
    table = torch.randn(100, 64, device="cuda", generator=gen(1)).bfloat16().requires_grad_()
    tokens, targets = tokens_of(30, 100, 1), targets_of(30, 64, 1)

    def loss(t):
        return ops.token_logprobs(ops.embedding(tokens, t), targets)[0].sum()

    alive = loss(table)  # its graph lives on
    want, = torch.autograd.grad(loss(table), table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaf = table.detach().clone().requires_grad_()
        torch.autograd.grad(loss(leaf), leaf)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got, = torch.autograd.grad(loss(leaf), leaf)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    again, = torch.autograd.grad(alive, table)
    assert torch.equal(again, want)
