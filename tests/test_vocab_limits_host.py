"""CPU: the widest rows that the embedding's gradient takes.  Columns are 32-bit numbers in its
kernels, with a slab of columns added to them."""
import pytest

from test_vocab_host import gradient

SHAPE = -2


@pytest.mark.parametrize("K", [(1 << 30) + 8, (1 << 31) - 2048, (1 << 31) - 1024, (1 << 31) - 8])
@pytest.mark.parametrize("T", [1, 5000])
def test_embedding_backward_refuses_wider_rows(nv, K, T):
    assert gradient(nv, K=K, ld=K, T=T, rows=1, n=1 << 60) == SHAPE
    assert nv.lib().nvfp4_embedding_backward_workspace_size(T, 1, K) == 0
