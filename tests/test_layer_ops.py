"""The torch.library operators of the 16-bit layers and the mixture of experts: schemas and
fake (shape) implementations on the CPU; on a GPU, autograd through a whole layer gives what
the direct calls give."""
import os
import subprocess
import sys

import pytest
import torch


def test_fake_shapes_without_a_gpu(nv):
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.nvfp4_b200
    with FakeTensorMode():
        x, w = torch.empty(30, 64, dtype=torch.bfloat16), torch.empty(4 * 96, 64, dtype=torch.bfloat16)
        offs = torch.empty(5, dtype=torch.int32)
        assert ops.linear(x, w).shape == (30, 384)
        assert ops.linear(x, w, offs, None, "swiglu").shape == (30, 48)
        y, z = ops.linear_preact(x, w, offs, None, "swiglu")
        assert y.shape == (30, 48) and z.shape == (30, 96) and y.dtype == torch.bfloat16
        r = ops.moe_route(torch.empty(15, 4), 2)
        assert [t.shape for t in r] == [(15, 2), (15, 2), (15, 2), (5,)] and r[0].dtype == torch.float32
        xs = ops.moe_dispatch(torch.empty(15, 64, dtype=torch.bfloat16), *r)
        assert xs.shape == (30, 64)
        assert ops.moe_combine(xs, *r).shape == (15, 64)


def test_preactivation_carries_no_gradient(nv):
    """linear_preact's z is not differentiable: a loss on it refuses instead of losing the
    term in silence."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.nvfp4_b200
    with FakeTensorMode():
        x = torch.empty(30, 64, dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(96, 64, dtype=torch.bfloat16, requires_grad=True)
        for act in ("silu", "swiglu", "none"):
            y, z = ops.linear_preact(x, w, None, None, act)
            assert y.requires_grad and not z.requires_grad
            with pytest.raises(RuntimeError, match="does not require grad"):
                z.float().square().sum().backward()
            gx, gw = torch.autograd.grad(y.sum(), [x, w])
            assert gx.shape == x.shape and gw.shape == w.shape


def test_bias_gradient_has_the_bias_shape(nv):
    """A dense layer takes its bias as [N] or [1, N] (one row of a grouped layer's)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.nvfp4_b200
    with FakeTensorMode():
        x, w = torch.empty(30, 64, dtype=torch.bfloat16), torch.empty(96, 64, dtype=torch.bfloat16)
        for offs, shape in ((None, (96,)), (None, (1, 96)), (torch.empty(2, dtype=torch.int32), (1, 96)),
                            (torch.empty(4, dtype=torch.int32), (3, 32))):
            b = torch.empty(shape, dtype=torch.bfloat16, requires_grad=True)
            y, _ = ops.linear_preact(x, w, offs, b, "silu")
            assert torch.autograd.grad(y.sum(), b)[0].shape == shape


def test_frozen_inputs_cost_no_gradient(nv):
    """The backward pass asks for the gradients that are wanted, no others."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.utils._python_dispatch import TorchDispatchMode
    ops, seen = torch.ops.nvfp4_b200, []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func is ops.linear_backward.default:
                seen.append([tuple(t.shape) for t in out])
            return out

    for wanted in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        with FakeTensorMode(), Log():
            x, w, b = (torch.empty(s, dtype=torch.bfloat16, requires_grad=bool(r))
                       for s, r in zip(((30, 64), (96, 64), (96,)), wanted))
            ops.linear_preact(x, w, None, b, "silu")[0].sum().backward()
            for t, r in zip((x, w, b), wanted):
                assert (t.grad is not None) == bool(r)
                assert not r or t.grad.shape == t.shape
        assert seen.pop() == [s if r else (0,) for s, r in zip(((30, 64), (96, 64), (96,)), wanted)]


@pytest.mark.gpu
def test_autograd_through_a_layer(nv, cuda_dev):
    ops = torch.ops.nvfp4_b200
    T, E, k, K, F, dt = 70, 8, 2, 64, 96, torch.bfloat16
    g = torch.Generator().manual_seed(3)

    def rnd(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to(dt).cuda().requires_grad_()

    x, wr = rnd(T, K), rnd(E, K, scale=0.1)
    w1, b1, w2 = rnd(E * 2 * F, K, scale=0.1), rnd(E, 2 * F, scale=0.1), rnd(E * K, F, scale=0.1)
    logits, _ = ops.linear_preact(x, wr)
    r = ops.moe_route(logits, k)
    xs = ops.moe_dispatch(x, *r)
    h, z = ops.linear_preact(xs, w1, r[3], b1, "swiglu")
    ys, _ = ops.linear_preact(h, w2, r[3])
    y = ops.moe_combine(ys, *r, x)
    dy = torch.randn(T, K, generator=g).to(dt).cuda()
    grads = torch.autograd.grad(y, [x, wr, w1, b1, w2], dy)

    with torch.no_grad():
        route = nv.Routing(*(t.detach() for t in r))
        dys, dwt = nv.moe_combine_backward(dy, ys.detach(), route)
        dh, dw2, _ = nv.linear_grouped_backward(dys, h.detach(), w2, route.m_offsets)
        dxs, dw1, db1 = nv.linear_grouped_backward(dh, xs.detach(), w1, route.m_offsets, preact=z, activation="swiglu",
                                                   bias_grad=True)
        dl = nv.moe_route_backward(dwt, logits.detach(), route)
        dxr, dwr, _ = nv.linear_backward(dl, x, wr)
        dx = dy.float() + nv.moe_dispatch_backward(dxs, route).float() + dxr.float()
    nv.device_status()
    for got, want in zip(grads[1:], (dwr, dw1, db1, dw2)):
        assert torch.equal(got, want)
    # three bf16 terms summed in bf16, in autograd's order: two roundings of at most 2^-8
    # of a partial sum, which is at most the sum of the terms' magnitudes
    size = dy.float().abs() + nv.moe_dispatch_backward(dxs, route).float().abs() + dxr.float().abs()
    assert ((grads[0].float() - dx).abs() <= 2.0 ** -7 * size).all()


GIL = """
import ctypes, sys, torch
sys.path.insert(0, "gpu-kernels_b200")
import nvfp4_b200 as nv
from nvfp4_b200 import _bind
from nvfp4_b200._lib import check
# every entry point answers whether its caller holds the GIL: 0 (no) is the good status
held = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
_bind._load().bind(check, *[held] * len(_bind._ENTRIES))
b, f = torch.bfloat16, torch.float32
x, w, l = torch.zeros(80, 64, dtype=b, device="cuda"), torch.zeros(64, 64, dtype=b, device="cuda"), \
    torch.zeros(80, 8, device="cuda")
i = torch.zeros(80, 1, dtype=torch.int32, device="cuda")
r = nv.Routing(torch.zeros(80, 1, device="cuda"), i, i, torch.zeros(9, dtype=torch.int32, device="cuda"))
for call in (lambda: nv.linear(x, w), lambda: nv.linear_backward(x, x, w, preact=x, activation="relu"),
             lambda: nv.moe_route(l, 2), lambda: nv.moe_route_backward(r.weights, l, r), lambda: nv.moe_dispatch(x, r),
             lambda: nv.moe_combine(x, r), lambda: nv.moe_combine_backward(x, x, r)):
    call()
print("done")
"""


@pytest.mark.gpu
def test_calls_release_the_gil(cuda_dev):
    """The library is called without the GIL, as through ctypes."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", GIL], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.stdout.strip() == "done", out.stderr[-2000:]
