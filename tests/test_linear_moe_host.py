"""CPU: what the 16-bit linear and mixture-of-experts entry points refuse, before any
device is touched."""
import ctypes as C

import pytest
import torch

P = C.c_void_p(1 << 20)    # never dereferenced: the checks run first
ODD = C.c_void_p((1 << 20) + 8)
INVALID, SHAPE, ALIGN, WORKSPACE = -1, -2, -3, -7


def linear(nv, X=P, ldx=64, W=P, bias=None, residual=None, Y=P, Z=None, offs=None, G=1, M=4, N=64, K=64, act=0, dt=0):
    return nv.lib().nvfp4_linear(X, ldx, W, bias, residual, Y, Z, offs, G, M, N, K, act, dt, None)


@pytest.mark.parametrize("args,status", [
    (dict(X=None), INVALID), (dict(W=None), INVALID), (dict(Y=None), INVALID), (dict(act=5), INVALID),
    (dict(act=-1), INVALID), (dict(dt=2), INVALID), (dict(G=0), INVALID), (dict(G=2), INVALID),
    (dict(M=-1), SHAPE), (dict(N=0), SHAPE), (dict(N=12), SHAPE), (dict(K=12, ldx=16), SHAPE), (dict(K=0), SHAPE),
    (dict(ldx=56), SHAPE), (dict(ldx=68), SHAPE), (dict(N=72, act=4), SHAPE), (dict(G=257, offs=P), SHAPE),
    (dict(X=ODD), ALIGN), (dict(W=ODD), ALIGN), (dict(Y=ODD), ALIGN), (dict(Z=ODD), ALIGN),
    (dict(residual=ODD), ALIGN), (dict(bias=C.c_void_p((1 << 20) + 1)), ALIGN),
    (dict(offs=C.c_void_p((1 << 20) + 2), G=2), ALIGN),
])
def test_linear_refusals(nv, args, status):
    assert linear(nv, **args) == status


def test_gradient_refusals(nv):
    L = nv.lib()
    assert L.nvfp4_linear_dgrad(None, P, P, None, 1, 4, 64, 64, 0, None) == INVALID
    assert L.nvfp4_linear_dgrad(P, P, P, None, 1, 4, 60, 64, 0, None) == SHAPE
    assert L.nvfp4_linear_dgrad(P, P, ODD, None, 1, 4, 64, 64, 0, None) == ALIGN
    assert L.nvfp4_linear_wgrad(P, P, 64, None, None, 1, 4, 64, 64, 0, None) == INVALID
    assert L.nvfp4_linear_wgrad(P, P, 32, P, None, 1, 4, 64, 64, 0, None) == SHAPE
    assert L.nvfp4_linear_wgrad(P, ODD, 64, P, None, 1, 4, 64, 64, 0, None) == ALIGN
    need = L.nvfp4_activation_backward_workspace_size(1, 100, 64)
    assert need > 0 and L.nvfp4_activation_backward_workspace_size(0, 100, 64) == 0
    assert L.nvfp4_activation_backward(P, P, P, P, None, 1, 100, 64, 1, 0, None, 0, None) == WORKSPACE
    assert L.nvfp4_activation_backward(P, P, P, P, None, 1, 100, 64, 1, 0, P, need - 1, None) == WORKSPACE
    assert L.nvfp4_activation_backward(P, None, P, None, None, 1, 100, 64, 1, 0, None, 0, None) == INVALID
    assert L.nvfp4_activation_backward(P, P, P, None, None, 1, 100, 48, 4, 0, None, 0, None) == SHAPE
    assert L.nvfp4_activation_backward(P, ODD, P, None, None, 1, 100, 64, 1, 0, None, 0, None) == ALIGN
    assert L.nvfp4_activation_backward(P, None, None, None, None, 1, 100, 64, 0, 0, None, 0, None) == 0  # nothing to do


def test_wide_tiles_hide_their_epilogue(nv):
    """A tile of two parts hides no epilogue under another tile: only where one round of the
    pairs takes all tiles, or a long reduction outweighs it and no round is lost."""
    import nvfp4_diag
    seen = set()
    for N, K in ((8192, 8192), (28672, 8192), (14344, 4104), (14336, 4096), (6144, 6144), (4096, 14336), (1024, 4096)):
        for M in (257, 300, 333, 450, 512, 1000, 1500, 3000, 4096, 8192, 16384):
            for form, features, red in (("forward", N, K), ("dgrad", K, N)):
                p = nvfp4_diag.linear_plan(form, M, N, K)
                if p["wide"]:
                    n_f, tiles = -(-features // 256), -(-M // p["bt"])
                    rounds = -(-(-(-tiles // 2) * n_f) // 74)
                    assert rounds == 1 or red > 199 * 64, (form, M, N, K)
                    seen.add(rounds == 1)
    assert seen == {True, False}
    assert nvfp4_diag.linear_plan("forward", 333, 14344, 4104)["wide"]
    assert nvfp4_diag.linear_plan("dgrad", 4096, 14336, 4096)["wide"]
    assert not nvfp4_diag.linear_plan("forward", 8192, 8192, 8192)["wide"]
    assert not nvfp4_diag.linear_plan("dgrad", 8192, 14336, 4096)["wide"]


def test_kernel_of_few_tokens(nv):
    """The choice where both kernels were measured: the faster one's, within 6 %.  Features,
    reduction, tokens, and the times (us) of the split-reduction and the persistent kernel."""
    import nvfp4_diag
    for form, features, red, M, split, persistent in (
            ("forward", 4096, 4096, 1, 9.9, 20.7), ("forward", 14336, 4096, 1, 22.8, 27.0),
            ("forward", 4096, 4096, 64, 15.8, 20.7), ("forward", 14336, 4096, 64, 24.8, 28.8),
            ("forward", 20480, 4096, 64, 34.1, 45.5), ("forward", 28672, 8192, 64, 79.9, 84.1),
            ("forward", 1024, 4096, 96, 10.6, 20.8), ("forward", 1024, 4096, 128, 12.3, 20.8),
            ("forward", 4096, 4096, 128, 21.2, 20.8), ("forward", 8192, 4096, 128, 23.4, 22.3),
            ("forward", 4096, 16384, 128, 37.3, 61.7), ("forward", 6144, 8192, 128, 30.1, 35.1),
            ("forward", 8192, 2048, 128, 17.6, 14.6), ("dgrad", 4096, 4096, 1, 12.5, 20.7),
            ("dgrad", 4096, 4096, 64, 18.6, 20.7), ("dgrad", 14336, 4096, 64, 26.9, 24.8),
            ("dgrad", 4096, 4096, 128, 24.8, 20.7), ("dgrad", 4096, 16384, 128, 39.7, 61.7),
            ("dgrad", 6144, 16384, 128, 48.2, 61.9)):
        n, k = (features, red) if form == "forward" else (red, features)
        chosen = split if nvfp4_diag.linear_plan(form, M, n, k)["decode"] else persistent
        assert chosen <= 1.06 * min(split, persistent), (form, features, red, M)


def test_extents_that_round_past_32_bits(nv):
    """The last 1023 sizes below 2^31 would round up past 32 bits inside the kernels."""
    big, L = (1 << 31) - 1, nv.lib()
    assert linear(nv, M=big) == SHAPE and linear(nv, N=big - 7, K=8) == SHAPE
    assert linear(nv, N=8, K=big - 7, ldx=big - 7) == SHAPE
    assert L.nvfp4_linear_dgrad(P, P, P, None, 1, big, 8, 8, 0, None) == SHAPE
    assert L.nvfp4_linear_wgrad(P, P, 8, P, None, 1, big, 8, 8, 0, None) == SHAPE
    assert L.nvfp4_activation_backward(P, P, P, None, None, 1, big, 8, 1, 0, None, 0, None) == SHAPE


def test_plan_of_many_tokens_is_quick(nv):
    """The host's choice of tiles takes as long for 2^31 tokens as for a few."""
    import time

    import nvfp4_diag
    nvfp4_diag.lib()
    t = time.perf_counter()
    for _ in range(100):
        p = nvfp4_diag.linear_plan("forward", (1 << 31) - 1024, 8, 4096)
    assert p["bt"] == 256 and time.perf_counter() - t < 0.1


def route(nv, logits=P, dt=0, bias=None, T=4, E=8, k=2, scoring=0, w=P, e=P, r=P, o=P, ws=None, n=0):
    return nv.lib().nvfp4_moe_route(logits, dt, bias, T, E, k, scoring, 1, 1.0, w, e, r, o, ws, n, None)


@pytest.mark.parametrize("args,status", [
    (dict(logits=None), INVALID), (dict(w=None), INVALID), (dict(e=None), INVALID), (dict(r=None), INVALID),
    (dict(o=None), INVALID), (dict(dt=3), INVALID), (dict(scoring=2), INVALID), (dict(bias=P), INVALID),
    (dict(T=-1), SHAPE), (dict(T=(1 << 20) + 1), SHAPE), (dict(E=0), SHAPE), (dict(E=257), SHAPE), (dict(k=0), SHAPE),
    (dict(k=9), SHAPE), (dict(E=64, k=33), SHAPE), (dict(logits=C.c_void_p((1 << 20) + 1)), ALIGN),
    (dict(logits=C.c_void_p((1 << 20) + 2), dt=2), ALIGN), (dict(T=129), WORKSPACE),
    (dict(T=129, ws=P, n=63), WORKSPACE),
])
def test_route_refusals(nv, args, status):
    assert route(nv, **args) == status


def test_move_refusals(nv):
    L = nv.lib()
    assert L.nvfp4_moe_route_workspace_size(129, 8) >= 64 and L.nvfp4_moe_route_workspace_size(5, 0) == 0
    assert L.nvfp4_moe_dispatch(None, P, P, 4, 8, 2, 64, P, None) == INVALID
    assert L.nvfp4_moe_dispatch(P, P, P, 4, 8, 2, 60, P, None) == SHAPE
    assert L.nvfp4_moe_dispatch(P, P, P, 4, 8, 33, 64, P, None) == SHAPE
    assert L.nvfp4_moe_dispatch(ODD, P, P, 4, 8, 2, 64, P, None) == ALIGN
    assert L.nvfp4_moe_combine(P, 2, P, P, None, 4, 2, 64, P, None) == INVALID
    assert L.nvfp4_moe_combine(P, 0, P, P, ODD, 4, 2, 64, P, None) == ALIGN
    assert L.nvfp4_moe_combine_backward(P, P, 0, P, None, P, 4, 8, 2, 64, P, P, None) == INVALID
    assert L.nvfp4_moe_combine_backward(P, P, 0, P, P, P, -1, 8, 2, 64, P, P, None) == SHAPE
    assert L.nvfp4_moe_route_backward(P, P, 0, None, 4, 8, 2, 0, 1, 1.0, P, None) == INVALID


def test_python_refuses_host_tensors(nv):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        nv.linear(x, w)
    with pytest.raises(ValueError):
        nv.moe_route(torch.zeros(4, 8), 2)
    r = nv.Routing(torch.zeros(4, 2), *(torch.zeros(4, 2, dtype=torch.int32) for _ in range(2)),
                   torch.zeros(9, dtype=torch.int32))
    with pytest.raises(ValueError):
        nv.moe_dispatch(x, r)


def test_gradients_are_launched_in_stream_order():
    """No kernel of the gradient is a programmatic dependent, the few-token input gradient
    included; the forward product of few tokens is one."""
    import nvfp4_diag
    seen = set()
    for M in (1, 16, 64, 128, 129, 1000):
        for N, K in ((8, 8), (4096, 4096), (8192, 512), (512, 8192), (14336, 4096)):
            for groups in (0, 1, 8):
                for form in ("dgrad", "wgrad"):
                    p = nvfp4_diag.linear_plan(form, M, N, K, groups)
                    assert not p["programmatic"], (form, M, N, K, groups)
                    seen.add((form, p["decode"]))
    assert ("dgrad", 1) in seen and ("dgrad", 0) in seen
    assert nvfp4_diag.linear_plan("forward", 1, 4096, 4096)["programmatic"]
