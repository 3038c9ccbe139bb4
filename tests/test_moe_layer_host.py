"""CPU: what the whole mixture-of-experts layer refuses, before any device is touched."""
import ctypes as C

import pytest
import torch

P = C.c_void_p(1 << 20)    # never dereferenced: the checks run first
ODD = C.c_void_p((1 << 20) + 8)
INVALID, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -7


def call(nv, x=P, ldx=64, logits=P, ldt=2, bias=None, w13=P, w2=P, residual=None, y=P, T=4, E=8, k=2, K=64, F=32,
         scoring=0, dt=0, ws=P, n=1 << 30):
    return nv.lib().nvfp4_moe_layer(x, ldx, logits, ldt, bias, w13, w2, residual, y, T, E, k, K, F, scoring, 1, 1.0, dt,
                                    ws, n, None)


@pytest.mark.parametrize("args,status", [
    (dict(x=None), INVALID), (dict(logits=None), INVALID), (dict(w13=None), INVALID), (dict(w2=None), INVALID),
    (dict(y=None), INVALID), (dict(dt=2), INVALID), (dict(ldt=3), INVALID), (dict(scoring=2), INVALID),
    (dict(bias=P), INVALID), (dict(T=-1), SHAPE), (dict(T=65), SHAPE), (dict(E=0), SHAPE), (dict(E=257), SHAPE),
    (dict(k=0), SHAPE), (dict(k=9), SHAPE), (dict(E=64, k=33), SHAPE), (dict(K=60), SHAPE), (dict(F=24), SHAPE),
    (dict(F=0), SHAPE), (dict(ldx=56), SHAPE), (dict(ldx=68), SHAPE), (dict(x=ODD), ALIGN), (dict(w13=ODD), ALIGN),
    (dict(w2=ODD), ALIGN), (dict(residual=ODD), ALIGN), (dict(y=ODD), ALIGN), (dict(ws=ODD), ALIGN),
    (dict(logits=C.c_void_p((1 << 20) + 2)), ALIGN), (dict(ws=None), WORKSPACE), (dict(n=1000), WORKSPACE),
])
def test_moe_layer_refusals(nv, args, status):
    assert call(nv, **args) == status


def test_moe_layer_workspace(nv):
    size = nv.lib().nvfp4_moe_layer_workspace_size
    assert size(0, 8, 2, 64, 32) == 0 and size(65, 8, 2, 64, 32) == 0 and size(4, 8, 2, 60, 32) == 0
    # hidden rows in 16 bits, the experts' results in 32, the routing
    assert size(16, 8, 2, 4096, 14336) >= 32 * (2 * 14336 + 4 * 4096 + 12)
    assert call(nv, n=size(4, 8, 2, 64, 32) - 1) == WORKSPACE


def test_python_refuses_host_tensors(nv):
    x, l = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 8)
    w13, w2 = torch.zeros(8 * 64, 64, dtype=torch.bfloat16), torch.zeros(8 * 64, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        nv.moe_layer(x, l, w13, w2, 2)
    with pytest.raises(ValueError):
        nv.moe_layer(x.repeat(20, 1), l.repeat(20, 1), w13, w2, 2)
