"""GPU: moe_layer refuses the same arguments whether its own kernels or the four operators it
stands for take the tokens."""
import pytest
import torch

from test_moe_layer_gpu import check, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [4, 64, 65, 130])
def test_moe_layer_refuses_whatever_the_tokens(nv, cuda_dev, T):
    E, K, F = 8, 64, 32
    d = layer(T, E, K, F, torch.bfloat16, 1)
    x, l, w13, w2 = d["x"], d["logits"], d["w13"], d["w2"]
    check(nv, d, 2)
    for call in (lambda: nv.moe_layer(x, l, w13, w2[:E * 56], 2), lambda: nv.moe_layer(x, l, w13, w2.repeat(2, 1), 2),
                 lambda: nv.moe_layer(x, l, w13, w2[:-1], 2), lambda: nv.moe_layer(x, l, w13[:-1], w2, 2),
                 lambda: nv.moe_layer(x, l, w13, w2[:, :24], 2), lambda: nv.moe_layer(x, l, w13, w2[:, :16].contiguous(), 2),
                 lambda: nv.moe_layer(x, l, w13[:E * F], w2, 2), lambda: nv.moe_layer(x, l, w13, w2[0], 2),
                 lambda: nv.moe_layer(x, l, w13, None, 2), lambda: nv.moe_layer(x, l, None, w2, 2),
                 lambda: nv.moe_layer(x, l, w13.half(), w2, 2), lambda: nv.moe_layer(x, l, w13, w2.half(), 2),
                 lambda: nv.moe_layer(x, l, w13.cpu(), w2, 2), lambda: nv.moe_layer(x, l, w13, w2.cpu(), 2),
                 lambda: nv.moe_layer(x.float(), l, w13, w2, 2), lambda: nv.moe_layer(x.cpu(), l, w13, w2, 2),
                 lambda: nv.moe_layer(x[:, :56], l, w13, w2, 2), lambda: nv.moe_layer(x, l[:3], w13, w2, 2),
                 lambda: nv.moe_layer(x, l.double(), w13, w2, 2), lambda: nv.moe_layer(x, l[0], w13, w2, 2),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, scoring="none"),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, bias=torch.zeros(E, device="cuda")),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, residual=x[:2]),
                 lambda: nv.moe_layer(x, l, w13, w2, 2, residual=x.float())):
        with pytest.raises(ValueError):
            call()
    for k in (0, 9):
        with pytest.raises(nv.NVFP4Error):
            nv.moe_layer(x, l, w13, w2, k)
    torch.cuda.synchronize()
    nv.device_status()
