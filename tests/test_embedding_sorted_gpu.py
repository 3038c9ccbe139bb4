"""GPU: the embedding's gradient by sorted tokens at the sizes of a training step: blocks of each
length, several slabs of columns, threads that a row's columns do not fill, tables larger than
what the sort zeroes; and the order of the sums, bit by bit, against a restatement on the CPU."""
import math

import numpy as np
import pytest
import torch

from test_vocab_gpu import check_embedding_backward, gen, tokens_of

pytestmark = pytest.mark.gpu


def normal(T, K, dtype, seed):
    return torch.randn(T, K, device="cuda", generator=gen(seed)).to(dtype)


# block of 32: up to 16384 tokens, or 512 columns; of 128: more than 32768 tokens of more than
# 1024 columns; of 64 between.  Slabs of 2048 columns.  The sort zeroes 144 MB of a table whose ids
# have up to 18 bits, 200 MB of one of up to 27; the joins 40 MB of the rest, the sums what is between.
SIZES = [(5000, 60000, 4096), (20000, 120000, 768), (17000, 90001, 1032), (33000, 40000, 2056), (40000, 30011, 4104),
         (33000, 150000, 1000), (70000, 200001, 520), (4097, 500000, 264), (9000, 70, 8200), (16385, 3, 1024),
         (32768, 45000, 2048), (32769, 45000, 2048), (131073, 1000, 1032)]


@pytest.mark.parametrize("T,rows,K", SIZES)
def test_embedding_backward_of_a_training_step(nv, cuda_dev, T, rows, K):
    dtype, index = (torch.bfloat16, torch.float16)[T % 2], (torch.int64, torch.int32)[rows % 2]
    dy = normal(T, K, dtype, T)
    t = tokens_of(T, rows, 1, index, 0.2, 0.1)
    dy[(t < 0) | (t >= rows)] = math.nan  # not read
    d = nv.embedding_backward(dy, t, rows, 0.5)
    dy = torch.nan_to_num(dy)
    assert torch.equal(d, check_embedding_backward(nv, dy, t, rows, 0.5))
    del d
    # one id for half the batch, at the end of the table, as a padding id may be; the others near it
    t = tokens_of(T, min(rows, 300), 2, torch.int64, 0.0, 0.0) + rows - min(rows, 300)
    t[torch.rand(T, device="cuda", generator=gen(3)) < 0.5] = rows - 1
    check_embedding_backward(nv, dy, t.to(index), rows, 2.0)


@pytest.mark.parametrize("T,rows,K", [(20000, 120000, 768), (4500, 200000, 512)])
def test_embedding_backward_every_row_named(nv, cuda_dev, T, rows, K):
    """Tokens in the rows that each launch zeroes, the first and the last of them among them: no
    zero is written over a sum."""
    dy = normal(T, K, torch.bfloat16, 5)
    row = K * 2
    edges = [0, 1]
    for done in ((32 << 20), (32 << 20) + (56 << 20), (32 << 20) + 2 * (56 << 20), rows * row - (40 << 20)):
        edges += [done // row + i for i in (-2, -1, 0, 1, 2)]
    edges += list(range(rows - 600, rows))
    t = torch.tensor([e for e in edges if 0 <= e < rows], device="cuda").repeat(T)[:T]
    t = t[torch.randperm(T, device="cuda", generator=gen(6))]
    check_embedding_backward(nv, dy, t, rows)


# ------------------------------------------------------------------------- the order of the sums
def cancelling(t, K, seed):
    """fp16 rows whose large parts cancel by pairs among each token's rows: what is left of a sum
    depends on its order, and shows in 16 bits.  fp16 [T, K] on the CPU."""
    g = torch.Generator().manual_seed(seed)
    out = torch.zeros(len(t), K)
    for v in t.unique():
        at = (t == v).nonzero()[:, 0]
        n = len(at) * 2 // 5
        big = torch.randn(n, K, generator=g) * 2.0 ** 11
        rows = torch.cat([big, -big, torch.randn(len(at) - 2 * n, K, generator=g)])
        out[at] = rows.gather(0, torch.rand(len(at), K, generator=g).argsort(0))
    return out.half()


def add_up(rows):
    s = np.zeros(rows.shape[1], np.float32)
    for r in rows:
        s = s + r
    return s


def restated(dy, t, rows, scale, block, few, reverse=False):
    """The documented order: equal tokens in the order of the batch.  Sorted: in blocks of the
    sorted order, in which tokens outside the table are last, and the blocks' sums one after
    another.  few: one after another up to 16 of them, more in eight pieces."""
    t = np.where((t < 0) | (t >= rows), rows, t)
    dy, order = dy.float().numpy(), np.argsort(t, kind="stable")
    if reverse:
        order = np.lexsort((-np.arange(len(t)), t))
    out = np.zeros((rows, dy.shape[1]), np.float32)
    sorted_t = t[order]
    for v in np.unique(sorted_t):
        if not 0 <= v < rows:
            continue
        at = np.flatnonzero(sorted_t == v)
        i0, n = at[0], len(at)
        if few:
            cuts = [n * w // 8 for w in range(9)] if n > 16 else [0, n]
        else:
            cuts = [0] + [c - i0 for c in range((i0 // block + 1) * block, i0 + n, block)] + [n]
        parts = [add_up(dy[order[i0 + a:i0 + b]]) for a, b in zip(cuts, cuts[1:])]
        s = parts[0]
        for p in parts[1:]:
            s = s + p
        out[v] = s
    return torch.from_numpy(out * np.float32(scale)).half()


@pytest.mark.parametrize("T,rows,K,block,few", [
    (2000, 40, 64, 0, True), (1500, 1, 520, 0, True), (3000, 7, 72, 0, True), (333, 9, 2056, 0, True),
    (9000, 5, 64, 32, False), (4200, 900, 264, 32, False), (6000, 1, 40, 32, False), (17000, 50, 520, 64, False),
    (17000, 3, 1032, 64, False), (33000, 400, 1032, 128, False)])
def test_embedding_backward_order_of_sums(nv, cuda_dev, T, rows, K, block, few):
    g = torch.Generator().manual_seed(K)
    t = torch.randint(-1, rows + 1, (T,), generator=g)
    t[torch.rand(T, generator=g) < 0.3] = rows // 2
    dy = cancelling(t, K, T)
    want = restated(dy, t.numpy(), rows, 0.5, block, few)
    # the inputs tell orders apart: in the reverse one the results are others
    assert (restated(dy, t.numpy(), rows, 0.5, block, few, reverse=True) != want).any()
    a = dy.cuda(), t.cuda()
    for _ in range(3):
        assert torch.equal(nv.embedding_backward(*a, rows, 0.5).cpu(), want)
