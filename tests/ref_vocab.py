"""Plain 64-bit forms of the embedding and of the token log probabilities, with error bounds
derived from the formats.

u is the unit roundoff of a 16-bit output (ref16.U), 2^-24 that of fp32.

Embedding gradient: n terms added one after another (and parts of them joined) in fp32 are off
by at most n 2^-24 times the sum of their absolute values; the product with the scale and the
final rounding follow.

Log probabilities.  With z = x / temperature and zm its row maximum:
  * log2(e) / temperature is two roundings (2^-23), a product and a subtraction fused one
    more: an exponent is off by at most 2^-22 |z - zm|, its power of two by 2^-22 more;
  * a thread adds V / 512 + 32 terms at most after another, all of one sign, and its sums are
    joined over at most 16 steps with a rescaling (2^-22) each;
  so the logarithm of the sum is off by at most
    e = (V / 512 + 32) 2^-24 + 16 2^-21 + 2^-22 (1 + E|z - zm|),  E over the probabilities,
  and a result adds a few roundings of itself and of what it is the difference of.
"""
import math

import torch

import ref16 as R

NONE = -math.inf


def embedding64(tokens, table, scale):
    t = tokens.reshape(-1).long()
    known = (t >= 0) & (t < table.shape[0])
    y = torch.zeros(t.numel(), table.shape[1], dtype=torch.float64, device=table.device)
    y[known] = table[t[known]].double() * scale
    return y.reshape(*tokens.shape, -1)


def embedding_backward64(dy, tokens, rows, scale):
    """(gradient, bound of its error before the rounding to 16 bits)."""
    t = tokens.reshape(-1).long()
    dy = dy.reshape(t.numel(), -1).double()
    known = (t >= 0) & (t < rows)
    d, a = (torch.zeros(rows, dy.shape[1], dtype=torch.float64, device=dy.device) for _ in range(2))
    n = torch.zeros(rows, dtype=torch.float64, device=dy.device)
    d.index_put_((t[known],), dy[known], accumulate=True)
    a.index_put_((t[known],), dy[known].abs(), accumulate=True)
    n.index_put_((t[known],), torch.ones_like(t[known], dtype=torch.float64), accumulate=True)
    return d * scale, (n[:, None] + 1) * 2.0 ** -24 * a * abs(scale)


class Logprobs:
    """One row after another in 64 bits; *_bound are the bounds above."""

    def __init__(self, logits, targets, V, k, temperature):
        x = logits[:, :V].double()
        x = torch.where(x.isnan(), torch.full_like(x, NONE), x)
        T = x.shape[0]
        z = x / temperature
        zm = z.amax(1)
        empty = zm == NONE
        ref = torch.where(empty, torch.zeros_like(zm), zm)
        e = torch.exp(z - ref[:, None])
        s = e.sum(1)
        self.lse = torch.where(empty, torch.full_like(s, NONE), ref + torch.log(s.clamp_min(1e-300)))
        # not z - lse: of rows at a type's lowest value even 64 bits keep nothing of log s there
        logp = (z - ref[:, None]) - torch.where(empty, torch.zeros_like(s), torch.log(s.clamp_min(1e-300)))[:, None]
        p = torch.where(empty[:, None], torch.zeros_like(e), e / s.clamp_min(1e-300)[:, None])
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        self.entropy = -plogp.sum(1)
        far = torch.where(p > 0, p * (ref[:, None] - z), torch.zeros_like(p)).sum(1)
        self.e = (V / 512 + 32) * 2.0 ** -24 + 16 * 2.0 ** -21 + 2.0 ** -22 * (1 + far)
        t = targets.long()
        self.known = (t >= 0) & (t < V)
        at = torch.where(self.known, t, torch.zeros_like(t))
        self.logprobs = torch.where(self.known, logp.gather(1, at[:, None])[:, 0], torch.zeros(()).double().to(x.device))
        self.logprobs = torch.where(self.known & empty, torch.full_like(self.logprobs, NONE), self.logprobs)
        size = lambda v: torch.where(v.isinf(), torch.zeros_like(v), v.abs())  # noqa: E731
        self.logprobs_bound = self.e + 2.0 ** -21 * (size(self.logprobs) + far + 1)
        self.lse_bound = self.e + 2.0 ** -21 * (size(ref) + size(self.lse))
        # S1 / S0: every term's own error and the sums', times E|z - zm|
        self.entropy_bound = 4 * self.e * (1 + far) + 2.0 ** -21 * (1 + self.entropy)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        live = x.gather(1, order) > NONE
        pad = k - order.shape[1]
        self.top_tokens = torch.nn.functional.pad(torch.where(live, order, torch.full_like(order, -1)), (0, pad), value=-1)
        top = torch.where(live, logp.gather(1, order), torch.full((), NONE, dtype=torch.float64, device=x.device))
        self.top_logprobs = torch.nn.functional.pad(top, (0, pad), value=NONE)
        self.p, self.logp, self.z, self.x, self.at, self.temperature = p, logp, z, x, at, temperature

    def grad(self, g, h, width):
        """(dlogits [T, width], bound)."""
        p, T = self.p, self.p.shape[0]
        g = torch.where(self.known, g.double(), torch.zeros_like(g, dtype=torch.float64))[:, None]
        h = torch.zeros_like(g) if h is None else h.double()[:, None]
        logp = torch.where(p > 0, self.logp, torch.zeros_like(p))
        d = -g * p - h * p * (logp + self.entropy[:, None])
        d = d.scatter_add(1, self.at[:, None], g)
        lse = torch.where(self.lse.isinf(), torch.zeros_like(self.lse), self.lse)
        z = torch.where(self.x > NONE, self.z, torch.zeros_like(self.z))
        r = 2.0 ** -21 * (z.abs() + lse.abs()[:, None] + 2) + self.lse_bound[:, None]  # of log p
        size = g.abs() + h.abs() * (logp.abs() + self.entropy[:, None])
        # an error r of log p makes p wrong by a factor e^r; once that is far from 1 all that is
        # left is that p and -p log p are between 0 and 1
        b = p * size * (torch.expm1(r.clamp_max(1)) + 2.0 ** -20) + p * h.abs() * (r + self.entropy_bound[:, None])
        b = torch.where(r < 0.5, b, g.abs() + h.abs() * (1 + self.entropy + self.entropy_bound)[:, None])
        # probabilities below 2^-126 are flushed to zero: at most so much of what they multiply
        b = b + 2.0 ** -126 * torch.where(p > 0, size, torch.zeros_like(size))
        b = b + 2.0 ** -22 * torch.zeros_like(b).scatter(1, self.at[:, None], g.abs())
        masked = ~(self.x > NONE)
        d, b = (torch.where(masked, torch.zeros_like(v), v) / self.temperature for v in (d, b))
        pad = (0, width - d.shape[1])
        return torch.nn.functional.pad(d, pad), torch.nn.functional.pad(b, pad)


def assert_near(got, ref, bound, what):
    """fp32 results; infinities have to be the same."""
    got, ref = got.double(), ref.double()
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    err, lim = (got[~inf] - ref[~inf]).abs(), bound.expand_as(ref)[~inf]
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} out of bounds, worst {(err - lim).max():.3e} above {lim.max():.3e}"


def assert_grad(got, ref, bound, what=""):
    if got.dtype == torch.float32:
        return assert_near(got, ref, bound + 2.0 ** -23 * ref.abs() + 1e-44, what)
    R.assert_close(got, ref, bound, what)
