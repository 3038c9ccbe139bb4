"""GPU: the largest tables that the embedding takes: offsets past 32 bits, counts at the end of int."""
import pytest
import torch

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
