"""GPU: token log probabilities where logits are large finite numbers: masks of -1e9 and the like,
rows at a mask alone, maxima far from zero; against the 64-bit forms and bounds of ref_vocab.py.
The rows go through each form of the kernel: a CTA's, a cluster's and a warp's."""
import math

import pytest
import torch

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
