"""GPU: the largest tables that the embedding takes: offsets past 32 bits, counts at the end of int."""
import pytest
import torch

import ref_vocab as V

pytestmark = pytest.mark.gpu
ROWS = 2 ** 31 - 1 - 1023  # the most there may be


@pytest.mark.parametrize("T", [3, 5000])
def test_embedding_of_the_most_rows(nv, cuda_dev, T):
    """34 GB of gradient, by tokens looked up by each other and sorted: every row is written, the
    last one too, and read back by the lookup."""
    K = 8
    t = torch.tensor([0, ROWS - 1, ROWS // 2], device="cuda")
    if T > 3:
        g = torch.Generator(device="cuda").manual_seed(1)
        t = torch.cat([t, torch.randint(0, ROWS, (T - 5,), device="cuda", generator=g),
                       torch.tensor([-1, ROWS], device="cuda")])
    t = t.to(torch.int32) if T == 3 else t
    dy = torch.ones(T, K, device="cuda", dtype=torch.bfloat16)
    d = nv.embedding_backward(dy, t, ROWS)
    try:
        nv.device_status()
        words = d.view(torch.int64).view(-1)  # two a row
        live = t[(t >= 0) & (t < ROWS)].long().unique()
        count = sum(int(torch.count_nonzero(words[i:i + (1 << 28)])) for i in range(0, words.numel(), 1 << 28))
        assert count == 2 * len(live)
        y = nv.embedding(t, d, 2.0)
        n = torch.stack([(t == v).sum() for v in t[:3]])
        assert torch.equal(y[:3].float(), (2.0 * n)[:, None].expand(3, K).float())
        assert (y[(t >= 0) & (t < ROWS)] >= 2).all() and not y[(t < 0) | (t >= ROWS)].any()
    finally:
        del d
        words = None
        torch.cuda.empty_cache()


@pytest.mark.parametrize("T,n,dtype", [(17000, 131072, torch.bfloat16), (300000, 8000, torch.float16),
                                       (17000, 131075, torch.float32)])
def test_logprobs_past_32_bits(nv, cuda_dev, T, n, dtype):
    """More logits than 2^31: the last rows are their own, and nothing else is written."""
    g = torch.Generator(device="cuda").manual_seed(2)
    block = (torch.randn(1000, n, device="cuda", generator=g) * 3).to(dtype)
    x = block.repeat(T // 1000, 1)
    x[-2:] = block[:2] + 1
    t = torch.randint(0, n, (T,), device="cuda", generator=g)
    dl, dh = torch.randn(T, device="cuda", generator=g), torch.randn(T, device="cuda", generator=g)
    try:
        r = nv.token_logprobs(x, t, None, 4, 0.7, True)
        pick = torch.tensor([0, 1, T // 2, (1 << 31) // n - 1, (1 << 31) // n, (1 << 31) // n + 1, T - 2, T - 1],
                            device="cuda")
        rows, at = x[pick].clone(), t[pick]
        ref = V.Logprobs(rows, at, n, 4, 0.7)
        V.assert_near(r.logprobs[pick], ref.logprobs, ref.logprobs_bound, "logprobs")
        V.assert_near(r.entropy[pick], ref.entropy, ref.entropy_bound, "entropy")
        assert torch.equal(r.top_tokens[pick].long(), ref.top_tokens)
        d = nv.token_logprobs_backward(dl, x, t, r, dh, None, 0.7, out=x)
        want, bound = ref.grad(dl[pick], dh[pick], n)
        V.assert_grad(d[pick], want, bound, "dlogits")
        nv.device_status()
    finally:
        x = d = None
        torch.cuda.empty_cache()


def test_embedding_past_32_bits(nv, cuda_dev):
    """More elements than 2^31 in the output, and in the gradient that comes in."""
    T, rows, K = 300000, 37, 8192
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn(rows, K, device="cuda", generator=g).bfloat16()
    t = torch.arange(T, device="cuda") % (rows + 1)  # the last is outside
    try:
        y = nv.embedding(t, table)
        for i in range(0, T, 50000):
            at = t[i:i + 50000]
            want = torch.where((at < rows)[:, None], table[at.clamp(max=rows - 1)], torch.zeros((), device="cuda").bfloat16())
            assert torch.equal(y[i:i + 50000], want)
        y[:-rows] = 0  # the last tokens alone count
        d = nv.embedding_backward(y, t, rows)
        last = t[-rows:]
        want = torch.zeros_like(table)
        want[last[last < rows]] = table[last[last < rows]]
        assert torch.equal(d, want)
        nv.device_status()
    finally:
        y = None
        torch.cuda.empty_cache()
