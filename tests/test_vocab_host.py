"""CPU: what the embedding and the token log probabilities refuse, and the 64-bit forms that
their GPU tests compare with, against autograd."""
import ctypes as C
import math

import pytest
import torch

import ref_vocab as V

P = C.c_void_p(1 << 20)    # never dereferenced: the checks run first
ODD = C.c_void_p((1 << 20) + 8)
TWO = C.c_void_p((1 << 20) + 2)
BYTE = C.c_void_p((1 << 20) + 1)
INVALID, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -7


def lookup(nv, tokens=P, tb=8, table=P, ld=64, scale=1.0, y=P, T=4, rows=100, K=64, dt=0):
    return nv.lib().nvfp4_embedding(tokens, tb, table, ld, scale, y, T, rows, K, dt, None)


@pytest.mark.parametrize("args,status", [
    (dict(tokens=None), INVALID), (dict(table=None), INVALID), (dict(y=None), INVALID), (dict(tb=2), INVALID),
    (dict(dt=2), INVALID), (dict(T=-1), SHAPE), (dict(rows=0), SHAPE), (dict(K=0), SHAPE), (dict(K=60), SHAPE),
    (dict(ld=56), SHAPE), (dict(ld=68), SHAPE), (dict(T=(1 << 31) - 1), SHAPE), (dict(rows=(1 << 31) - 1), SHAPE),
    (dict(T=1 << 30, K=1 << 20, ld=1 << 20), SHAPE), (dict(tokens=C.c_void_p((1 << 20) + 4)), ALIGN),
    (dict(tokens=TWO, tb=4), ALIGN), (dict(table=ODD), ALIGN), (dict(y=ODD), ALIGN),
])
def test_embedding_refusals(nv, args, status):
    assert lookup(nv, **args) == status


def gradient(nv, dy=P, ld=64, tokens=P, tb=8, d=P, T=4, rows=100, K=64, dt=0, ws=P, n=1 << 30):
    return nv.lib().nvfp4_embedding_backward(dy, ld, tokens, tb, 1.0, d, T, rows, K, dt, ws, n, None)


@pytest.mark.parametrize("args,status", [
    (dict(dy=None), INVALID), (dict(tokens=None), INVALID), (dict(d=None), INVALID), (dict(tb=1), INVALID),
    (dict(dt=2), INVALID), (dict(T=-1), SHAPE), (dict(rows=0), SHAPE), (dict(K=12), SHAPE), (dict(ld=60), SHAPE),
    (dict(dy=ODD), ALIGN), (dict(d=ODD), ALIGN), (dict(ws=ODD), ALIGN), (dict(ws=None, n=0, T=5000), WORKSPACE),
    (dict(n=100, T=5000), WORKSPACE),
])
def test_embedding_backward_refusals(nv, args, status):
    assert gradient(nv, **args) == status


def test_embedding_workspace(nv):
    size = nv.lib().nvfp4_embedding_backward_workspace_size
    assert size(0, 100, 64) == 0 and size(4, 0, 64) == 0 and size(4, 100, 4) == 0
    assert size(2048, 1 << 17, 4096) == size(4096, 1 << 17, 64) == 0  # few tokens are not sorted
    last = 0
    for T in (4096, 4097, 32768, 32769, 131073, 1 << 20, 1 << 24):
        n = size(T, 1 << 17, 4096)
        assert n >= 16 * T and n % 256 == 0
        last = n
    assert last < 1 << 40


def forward(nv, x=P, ld=100, dt=0, t=P, tb=8, T=4, vocab=100, k=0, temp=1.0, lp=P, ent=None, top=None, tok=None, lse=P):
    return nv.lib().nvfp4_token_logprobs(x, ld, dt, t, tb, T, vocab, k, temp, lp, ent, top, tok, lse, None)


@pytest.mark.parametrize("args,status", [
    (dict(x=None), INVALID), (dict(t=None), INVALID), (dict(lp=None), INVALID), (dict(lse=None), INVALID),
    (dict(dt=3), INVALID), (dict(dt=-1), INVALID), (dict(tb=2), INVALID), (dict(temp=0.0), INVALID),
    (dict(temp=-1.0), INVALID), (dict(temp=math.inf), INVALID), (dict(temp=math.nan), INVALID),
    (dict(temp=1e-39), INVALID), (dict(k=3), INVALID), (dict(k=3, top=P), INVALID), (dict(k=-1), SHAPE),
    (dict(k=33, top=P, tok=P), SHAPE), (dict(T=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(ld=99), SHAPE),
    (dict(vocab=(1 << 31) - 1, ld=1 << 40), SHAPE), (dict(x=BYTE), ALIGN), (dict(x=TWO, dt=2), ALIGN),
    (dict(t=TWO, tb=4), ALIGN), (dict(t=C.c_void_p((1 << 20) + 4)), ALIGN), (dict(lp=TWO), ALIGN),
    (dict(ent=TWO), ALIGN), (dict(lse=TWO), ALIGN), (dict(k=1, top=TWO, tok=P), ALIGN),
    (dict(k=1, top=P, tok=TWO), ALIGN),
])
def test_logprobs_refusals(nv, args, status):
    assert forward(nv, **args) == status


def backward(nv, g=P, h=None, x=P, ld=100, dt=0, t=P, tb=8, lse=P, ent=None, T=4, vocab=90, W=100, temp=1.0, d=P,
             ldd=100):
    return nv.lib().nvfp4_token_logprobs_backward(g, h, x, ld, dt, t, tb, lse, ent, T, vocab, W, temp, d, ldd, None)


@pytest.mark.parametrize("args,status", [
    (dict(g=None), INVALID), (dict(x=None), INVALID), (dict(t=None), INVALID), (dict(lse=None), INVALID),
    (dict(d=None), INVALID), (dict(h=P), INVALID), (dict(dt=3), INVALID), (dict(tb=0), INVALID),
    (dict(temp=0.0), INVALID), (dict(T=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(W=89), SHAPE), (dict(ld=99), SHAPE),
    (dict(ldd=99), SHAPE), (dict(T=1 << 30, W=1 << 20, ld=1 << 20, ldd=1 << 20), SHAPE), (dict(x=BYTE), ALIGN),
    (dict(d=BYTE), ALIGN), (dict(d=TWO, dt=2), ALIGN), (dict(g=TWO), ALIGN), (dict(h=TWO, ent=P), ALIGN),
    (dict(h=P, ent=TWO), ALIGN), (dict(lse=TWO), ALIGN),
])
def test_logprobs_backward_refusals(nv, args, status):
    assert backward(nv, **args) == status


def test_python_refuses_host_tensors(nv):
    tokens, table = torch.zeros(4, dtype=torch.int64), torch.zeros(8, 64, dtype=torch.bfloat16)
    logits = torch.zeros(4, 64)
    result = nv.TokenLogprobs(torch.zeros(4), None, None, None, torch.zeros(4))
    for call in (lambda: nv.embedding(tokens, table), lambda: nv.embedding_backward(table[:4], tokens, 8),
                 lambda: nv.token_logprobs(logits, tokens),
                 lambda: nv.token_logprobs_backward(torch.zeros(4), logits, tokens, result)):
        with pytest.raises(ValueError):
            call()


def test_reference_gradients():
    """The 64-bit forms are their own gradients' primitives."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 12, generator=g, dtype=torch.float64) * 3
    x[1, 3:9] = -math.inf
    targets = torch.tensor([0, 2, -1, 9, 40])
    a, b = torch.randn(5, generator=g, dtype=torch.float64), torch.randn(5, generator=g, dtype=torch.float64)
    r = V.Logprobs(x, targets, 10, 3, 0.7)
    d, _ = r.grad(a, b, 12)
    leaf = x.clone().requires_grad_()
    lp = torch.log_softmax(leaf[:, :10] / 0.7, 1)
    h = -(lp.exp() * lp.masked_fill(lp == -math.inf, 0.0)).sum(1)
    mine = torch.stack([lp[t, v] if 0 <= v < 10 else torch.zeros((), dtype=torch.float64)
                        for t, v in enumerate(targets.tolist())])
    assert torch.allclose(r.logprobs, mine.detach()) and torch.allclose(r.entropy, h.detach())
    want, = torch.autograd.grad((mine * a).sum() + (h * b).sum(), leaf)
    assert torch.allclose(d, torch.nan_to_num(want), atol=1e-12)
    dy = torch.randn(6, 8, generator=g, dtype=torch.float64)
    tokens = torch.tensor([[3, 0, 3], [-1, 9, 3]])
    table = torch.zeros(5, 8, dtype=torch.float64, requires_grad=True)
    y = V.embedding64(tokens, table.detach(), 2.0)
    assert y.shape == (2, 3, 8)
    d, _ = V.embedding_backward64(dy.reshape(2, 3, 8), tokens, 5, 2.0)
    assert torch.allclose(d[3], 2 * (dy[0] + dy[2] + dy[5])) and torch.allclose(d[0], 2 * dy[1]) and not d[1].any()
