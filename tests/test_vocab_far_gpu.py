"""GPU: token log probabilities where logits are large finite numbers: masks of -1e9 and the like,
rows at a mask alone, maxima far from zero; against the 64-bit forms and bounds of ref_vocab.py.
The rows go through each form of the kernel: a CTA's, a cluster's and a warp's."""
import math

import pytest
import torch

import ref_vocab as V
from test_vocab_gpu import check_logprobs, gen

pytestmark = pytest.mark.gpu

# rows and vocabulary by the form that takes them on 148 SMs: a CTA a row (more rows than half the
# SMs), a cluster a row (few long rows), a warp a row (short rows, more than three an SM)
FORMS = {"cta": (160, 9001), "cluster": (9, 70001), "warp": (1000, 3001)}


def far_rows(form, dtype, mask, seed=0):
    """(logits, targets): row kinds in turn; the target is a live token, a masked one or ignored."""
    T, n = FORMS[form]
    g = gen(seed)
    mask = max(mask, torch.finfo(dtype).min)
    x = torch.randn(T, n, device="cuda", generator=g) * 3
    live = torch.randint(0, n, (T,), device="cuda", generator=g)
    row = torch.arange(T, device="cuda")
    kind = row % 9
    half = torch.rand(T, n, device="cuda", generator=g) < 0.5
    x = torch.where((kind == 0)[:, None] | ((kind == 1)[:, None] & half) | (kind == 2)[:, None], mask, x)
    x[kind == 3, : n // 2] = mask                  # first parts, batches and vectors of masks alone
    x[kind == 4, n // 3:] = mask
    x[kind == 5, 1:] = x[kind == 5, 1:] + mask     # at the mask, spread where the type can
    x[row[(kind == 0) | (kind == 5)], live[(kind == 0) | (kind == 5)]] = 2.0
    x[kind == 6, ::7] = -math.inf                  # both sorts of mask
    x[kind == 6, 3::7] = mask
    high = row[(kind == 7) | (kind == 8)]
    x[high, live[high]] = -mask                    # one maximum far above, or two equal ones
    x[kind == 8, 5] = -mask
    t = live.clone()
    t[row % 4 == 1] = (live[row % 4 == 1] + 11) % n
    t[row % 11 == 10] = -100
    return x.to(dtype), t


MASKS = [(torch.bfloat16, m) for m in (-1e9, -1e10, -1e12, -1e15)]
MASKS += [(torch.float32, m) for m in (-1e9, -1e10, -1e12, -1e15)]
MASKS += [(torch.float16, m) for m in (-1e4, -65504.0)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_logprobs_large_logits(nv, cuda_dev, form, dtype, mask):
    x, t = far_rows(form, dtype, mask)
    for i, temperature in enumerate((1.0, 0.5, 0.3, 0.1, 2.5, 1e-3)):
        r = check_logprobs(nv, x, t, None, (0, 5)[i % 2], temperature)
        assert torch.isfinite(r.lse).all() and torch.isfinite(r.entropy).all() and not r.logprobs.isnan().any()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_one_value_alone(nv, cuda_dev, form, dtype):
    """Rows of one value of any size: log probability -ln n, entropy ln n."""
    T, n = FORMS[form]
    x = torch.zeros(T, n, device="cuda")
    at = torch.arange(T, device="cuda")
    sign = torch.where(at % 2 == 0, 1.0, -1.0)
    x += (sign * 10.0 ** (at % 37).float())[:, None]  # 1 to 1e36
    x = x.to(dtype)
    t = at % n
    r = check_logprobs(nv, x, t, None, 3, grad=False)
    # the sum of n equal terms in fp32: the bound of ref_vocab without a difference to the maximum
    e = (n / 512 + 32) * 2.0 ** -24 + 16 * 2.0 ** -21 + 2.0 ** -21 * (1 + math.log(n))
    assert (r.logprobs.double() + math.log(n)).abs().max() <= e
    assert (r.entropy.double() - math.log(n)).abs().max() <= 4 * e + 2.0 ** -21 * (1 + math.log(n))
    assert (r.top_tokens == torch.arange(3, device="cuda")).all()


# ------------------------------------------------------------------------- gradient
def grad64(ref, g, h, width, limit):
    """(dlogits, bound).  Where |lse| is at most `limit` the probabilities come from lse, and the
    bound is ref_vocab's; beyond it log p = (z - zm) - ln s, of the row's own maximum and sum: off
    by ln s's error, which is `e` of ref_vocab, and by a few roundings of z - zm, however large z is."""
    want, near = ref.grad(g, h, width)
    g = torch.where(ref.known, g.double(), torch.zeros_like(g, dtype=torch.float64))[:, None]
    h = torch.zeros_like(g) if h is None else h.double()[:, None]
    p, logp = ref.p, torch.where(ref.p > 0, ref.logp, torch.zeros_like(ref.p))
    zm = torch.where(ref.lse.isinf(), torch.zeros_like(ref.lse), ref.z.amax(1))[:, None]
    z = torch.where(ref.x > -math.inf, ref.z, zm)
    r = ref.e[:, None] + 2.0 ** -21 * (zm - z + 1)
    size = g.abs() + h.abs() * (logp.abs() + ref.entropy[:, None])
    b = p * size * (torch.expm1(r.clamp_max(1)) + 2.0 ** -20) + p * h.abs() * (r + ref.entropy_bound[:, None])
    b = b + 2.0 ** -126 * torch.where(p > 0, size, torch.zeros_like(size))
    b = b + 2.0 ** -22 * torch.zeros_like(b).scatter(1, ref.at[:, None], g.abs())
    b = torch.where(ref.x > -math.inf, b, torch.zeros_like(b)) / ref.temperature
    b = torch.nn.functional.pad(b, (0, width - b.shape[1]))
    return want, torch.where((ref.lse.abs() <= limit)[:, None], near, b)


def check_gradient(nv, x, t, vocab=None, temperature=1.0, out=None):
    n = x.shape[1] if vocab is None else vocab
    r = nv.token_logprobs(x, t, vocab, 0, temperature, True)
    ref = V.Logprobs(x, t, n, 0, temperature)
    rand = gen(7)
    dl, dh = torch.randn(len(t), device="cuda", generator=rand), torch.randn(len(t), device="cuda", generator=rand)
    limit = 64.0 if x.dtype == torch.float32 else 256.0
    for h in (None, dh):
        want, bound = grad64(ref, dl, h, x.shape[1], limit)
        d = nv.token_logprobs_backward(dl, x, t, r, h, vocab, temperature, out)
        # what lies past the type's largest number rounds to infinity
        most = torch.finfo(x.dtype).max
        past = want.abs() - bound > most
        assert (d[past].double() * want[past].sign() >= 0.99 * most).all()
        skip = past | (d.isinf() & (want.abs() + bound > most))
        V.assert_grad(*(torch.where(skip, torch.zeros_like(v), v) for v in (d, want, bound)), "dlogits")
    own = x.clone()
    assert torch.equal(nv.token_logprobs_backward(dl, own, t, r, dh, vocab, temperature, out=own), d)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_logprobs_gradient_of_large_logits(nv, cuda_dev, form, dtype, mask):
    x, t = far_rows(form, dtype, mask)
    for temperature in (1.0, 0.3, 1e-3):
        check_gradient(nv, x, t, None, temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,vocab,W", [(5, 1, 1), (7, 7, 9), (300, 40, 40), (9, 1000, 1003), (33, 2040, 2056),
                                       (20, 4001, 4001), (6, 9001, 9004), (3, 70001, 70001)])
def test_logprobs_gradient_far_from_zero(nv, cuda_dev, dtype, T, vocab, W):
    """Logits around a large number, and small temperatures: log sum exp is large in both."""
    x = torch.randn(T, W, device="cuda", generator=gen(W)) * 3
    shift = torch.tensor([0.0, 60.0, -70.0, 250.0, -300.0, 3000.0, -2e4], device="cuda").repeat(T // 7 + 1)[:T]
    x = (x + shift[:, None]).to(dtype)
    x[T // 2, ::3] = -math.inf
    t = torch.randint(0, vocab, (T,), device="cuda", generator=gen(1))
    t[T // 3] = -1
    for temperature in (1.0, 0.05, 1e-3, 1e-5, 1e-20):
        check_gradient(nv, x, t, vocab, temperature)
    wide = torch.empty(T, W + 9, device="cuda", dtype=dtype)
    check_gradient(nv, x, t, vocab, 0.01, out=wide[:, 3:3 + W])


def test_logprobs_gradient_of_masked_rows_is_shared(nv, cuda_dev):
    """A row wholly at a mask is uniform: -g / n beside the target."""
    for n in (100, 5000):
        for value in (-1e10, -1e30, 1e10, 1e4):
            x = torch.full((3, n), value, device="cuda")
            t = torch.tensor([0, 50, 99], device="cuda")
            r = nv.token_logprobs(x, t)
            d = nv.token_logprobs_backward(torch.ones(3, device="cuda"), x, t, r).double()
            want = torch.full_like(d, -1 / n).scatter_add_(1, t[:, None], torch.ones_like(d))
            assert (d - want).abs().max() <= 2.0 ** -20
