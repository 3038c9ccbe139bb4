"""The 16-bit linear layers on the GPU against 64-bit forms, within bounds derived from the
number formats (ref16.py): tile edges, ragged and empty groups, strides, activations, and
gradients against the formula and against differences."""
import math

import pytest
import torch

import ref16 as R

pytestmark = pytest.mark.gpu


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def offsets(cuts):
    return torch.tensor(cuts, dtype=torch.int32, device="cuda")


def check_forward(nv, M, N, K, act="none", bias=False, residual=False, dtype=torch.bfloat16, cuts=None, z=False):
    G = 1 if cuts is None else len(cuts) - 1
    x, w = make((M, K), dtype, 1), make((G * N, K), dtype, 2, K ** -0.5)
    b = make((N,) if cuts is None else (G, N), dtype, 3, 0.5) if bias else None
    No = N // 2 if act == "swiglu" else N
    r = make((M, No), dtype, 4) if residual else None
    if cuts is None:
        got = nv.linear(x, w, bias=b, activation=act, residual=r, return_preact=z)
    else:
        got = nv.linear_grouped(x, w, offsets(cuts), bias=b, activation=act, return_preact=z)
    nv.device_status()
    y, ey, zz, ez = R.forward64(x, w, cuts or [0, M], b, act, r)
    if z:
        R.assert_close(got[1], zz, ez, "z")
        got = got[0]
    R.assert_close(got, y, ey, "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [
    (1, 8, 8), (1, 256, 64), (2, 264, 72), (15, 512, 128), (16, 248, 200), (17, 1024, 1032), (31, 128, 64),
    (33, 320, 456), (64, 4096, 512), (65, 264, 2048), (127, 256, 264), (128, 2048, 1024), (129, 520, 128),
    (200, 1000, 640), (256, 256, 4096), (257, 768, 64), (300, 2056, 96), (513, 264, 8), (1025, 1288, 520),
])
def test_shapes(nv, cuda_dev, M, N, K, dtype):
    check_forward(nv, M, N, K, dtype=dtype)


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("M,N,K", [(1, 512, 256), (5, 288, 136), (48, 1056, 512), (130, 544, 264), (700, 1312, 192)])
def test_epilogue(nv, cuda_dev, act, M, N, K):
    for dtype in (torch.bfloat16, torch.float16):
        check_forward(nv, M, N, K, act, bias=True, residual=True, dtype=dtype, z=True)
        check_forward(nv, M, N, K, act, bias=True, dtype=dtype)
        check_forward(nv, M, N, K, act, residual=True, dtype=dtype)


GROUPS = [
    [0, 5], [0, 0, 3, 3, 40], [0, 1, 2, 3, 4, 5], [0, 17, 17, 50, 300], [0, 256, 512, 700], [0, 300, 301, 301, 557, 900],
    [0] * 20 + [9], [0, 33, 66, 99, 132, 165, 198], list(range(0, 65 * 8, 8)),
]


@pytest.mark.parametrize("cuts", GROUPS, ids=lambda c: f"G{len(c) - 1}M{c[-1]}")
def test_groups(nv, cuda_dev, cuts):
    check_forward(nv, cuts[-1], 264, 136, cuts=cuts)
    check_forward(nv, cuts[-1], 544, 200, "swiglu", bias=True, cuts=cuts, z=True, dtype=torch.float16)
    check_forward(nv, cuts[-1], 256, 512, "gelu_tanh", bias=True, cuts=cuts)


def plan(form, M, N, K, groups=0):
    import nvfp4_diag
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return nvfp4_diag.linear_plan(form, M, N, K, groups, sms)


@pytest.mark.parametrize("act", R.ACTS)
def test_wide_tiles(nv, cuda_dev, act):
    """Tiles of two parts: ends in the first part, in the second, and full ones."""
    for M, N, K, dtype, residual in ((257, 14368, 2056, torch.bfloat16, True), (333, 14368, 2056, torch.float16, False),
                                     (385, 14368, 2056, torch.float16, True), (450, 14368, 4104, torch.bfloat16, True),
                                     (512, 14368, 4104, torch.bfloat16, False)):
        p = plan("forward", M, N, K)
        assert p["wide"] and p["bt"] < M <= 2 * p["bt"]
        check_forward(nv, M, N, K, act, bias=True, residual=residual, dtype=dtype, z=True)


@pytest.mark.parametrize("M,dtype", [(257, torch.bfloat16), (333, torch.float16), (450, torch.bfloat16)])
def test_wide_tiles_input_gradient(nv, cuda_dev, M, dtype):
    N, K = 4104, 14344
    assert plan("dgrad", M, N, K)["wide"]
    x, w, dy = make((M, K), dtype, 1), make((N, K), dtype, 2, K ** -0.5), make((M, N), dtype, 3)
    z = make((M, N), dtype, 4)
    dx, _, db = nv.linear_backward(dy, x, w, preact=z, activation="silu", bias_grad=True, weight_grad=False)
    nv.device_status()
    ref = R.backward64(dy, x, w, [0, M], z, "silu")
    R.assert_close(dx, *ref[0], "dx")
    R.assert_close(db, *(t.flatten() for t in ref[2]), "db")


def test_wide_tiles_in_rounds(nv, cuda_dev):
    """Wide tiles one after the other on a pair (a long reduction), forward and input gradient."""
    for form, M, N, K in (("forward", 700, 14344, 12808), ("dgrad", 1550, 12808, 6152)):
        p = plan(form, M, N, K)
        assert p["wide"] and -(-M // (2 * p["bt"])) * -(-(N if form == "forward" else K) // 256) > 74
    check_forward(nv, 700, 14344, 12808, "silu", bias=True, residual=True, dtype=torch.float16, z=True)
    M, N, K = 1550, 12808, 6152
    x, w, dy = make((M, K), torch.bfloat16, 1), make((N, K), torch.bfloat16, 2, N ** -0.5), make((M, N), torch.bfloat16, 3)
    dx = nv.linear_backward(dy, x, w, weight_grad=False)[0]
    nv.device_status()
    ref = dy.double() @ w.double()
    R.assert_close(dx, ref, R.acc(N) * (dy.double().abs() @ w.double().abs()), "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 512, 8200), (16, 264, 16384), (64, 512, 8200), (100, 520, 8200), (128, 512, 8200)])
def test_few_tokens_long_reduction(nv, cuda_dev, M, N, K, dtype):
    """The split-reduction kernel where its ring goes round and eight CTAs share a tile, forward
    and (with N and K exchanged) input gradient, up to its most tokens."""
    for form, n, k in (("forward", N, K), ("dgrad", K, N)):
        p = plan(form, M, n, k)
        assert p["decode"] and p["splits"] == 8 and -(-K // 64) // 8 > p["stages"]
    check_forward(nv, M, N, K, "silu", bias=True, residual=True, dtype=dtype, z=True)
    if N % 32 == 0:
        check_forward(nv, M, N, K, "swiglu", bias=True, residual=True, dtype=dtype, z=True)
    x, w, dy = make((M, N), dtype, 1), make((K, N), dtype, 2, K ** -0.5), make((M, K), dtype, 3)
    dx, dw, _ = nv.linear_backward(dy, x, w)
    nv.device_status()
    for got, (r, e), n in zip((dx, dw), R.backward64(dy, x, w, [0, M], None, "none"), ("dx", "dw")):
        R.assert_close(got, r, e, n)


def test_few_tokens_long_reduction_by_groups(nv, cuda_dev):
    cuts = [0, 3, 3, 20, 21, 40]
    M, N, K = cuts[-1], 264, 8200
    for form, n, k in (("forward", N, K), ("dgrad", K, N)):
        p = plan(form, M, n, k, len(cuts) - 1)
        assert p["decode"] and p["splits"] == 8 and -(-K // 64) // 8 > p["stages"]
    check_forward(nv, M, N, K, "relu", bias=True, cuts=cuts, z=True)
    G = len(cuts) - 1
    x, w, dy = make((M, N), torch.bfloat16, 1), make((G * K, N), torch.bfloat16, 2, K ** -0.5), make((M, K), torch.bfloat16, 3)
    dx = nv.linear_grouped_backward(dy, x, w, offsets(cuts), weight_grad=False)[0]
    nv.device_status()
    R.assert_close(dx, *R.backward64(dy, x, w, cuts, None, "none")[0], "dx")


@pytest.mark.parametrize("bt,M,N,K", [(64, 130, 264, 72), (96, 450, 9480, 72), (128, 200, 6152, 520),
                                      (160, 130, 14368, 520), (192, 333, 6152, 1032), (224, 200, 14368, 1032),
                                      (256, 500, 14368, 520)])
def test_every_tile_width(nv, cuda_dev, bt, M, N, K):
    p = plan("forward", M, N, K)
    assert not p["decode"] and p["bt"] == bt and not p["wide"]
    check_forward(nv, M, N, K, bias=True)


def test_rows_outside_groups_are_zero(nv, cuda_dev):
    """Offsets that leave rows out at both ends, and ends past the last row (clamped)."""
    x, w = make((300, 128), torch.bfloat16, 1), make((2 * 64, 128), torch.bfloat16, 2)
    y, z = nv.linear_grouped(x, w, offsets([7, 100, 250]), activation="silu", return_preact=True)
    ref, e, zr, ez = R.forward64(x, w, [7, 100, 250], None, "silu", None)
    R.assert_close(y, ref, e)
    R.assert_close(z, zr, ez)
    assert not y[:7].any() and not y[250:].any() and not z[:7].any() and not z[250:].any()
    y = nv.linear_grouped(x, w, offsets([-5, 100, 5000]))
    R.assert_close(y, *R.forward64(x, w, [0, 100, 300], None, "none", None)[:2])
    y = nv.linear_grouped(x, w, offsets([0, 0, 0]))
    assert not y.any()


def test_empty(nv, cuda_dev):
    w = make((64, 32), torch.bfloat16, 2)
    x = w.new_empty((0, 32))
    assert nv.linear(x, w).shape == (0, 64)
    dx, dw, db = nv.linear_backward(x.new_empty((0, 64)), x, w, bias_grad=True)
    assert dx.shape == (0, 32) and not dw.any() and not db.any()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_strided_rows(nv, cuda_dev, M):
    """x as a slice of wider rows, whose other columns hold NaN."""
    wide = torch.full((M, 512), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, 64:64 + 136] = make((M, 136), torch.bfloat16, 1)
    x, w = wide[:, 64:64 + 136], make((264, 136), torch.bfloat16, 2)
    R.assert_close(nv.linear(x, w), *R.forward64(x, w, [0, M], None, "none", None)[:2])
    dy = make((M, 264), torch.bfloat16, 3)
    _, dw, _ = nv.linear_backward(dy, x, w)
    (_, _), (ref, e), _ = R.backward64(dy, x, w, [0, M], None, "none")
    R.assert_close(dw, ref, e)


def test_one_row_of_any_stride(nv, cuda_dev):
    """The stride of a single row does not matter, whatever it is."""
    w, dy = make((264, 136), torch.bfloat16, 2), make((1, 264), torch.bfloat16, 3)
    for cols in (137, 4099):
        x = make((2, cols), torch.bfloat16, 1)[:1, :136]
        assert x.stride(0) == cols
        R.assert_close(nv.linear(x, w), *R.forward64(x, w, [0, 1], None, "none", None)[:2])
        for got, (r, e) in zip(nv.linear_backward(dy, x, w)[:2], R.backward64(dy, x, w, [0, 1], None, "none")):
            R.assert_close(got, r, e)


def test_other_groups_values_stay_out(nv, cuda_dev):
    """Infinities and NaN in another group's rows and weights reach only that group."""
    cuts = [0, 21, 40, 73]
    x, w, dy = make((73, 72), torch.bfloat16, 1), make((3 * 72, 72), torch.bfloat16, 2), make((73, 72), torch.bfloat16, 3)
    clean = [t.clone() for t in (x, w, dy)]
    for t, rows in ((x, slice(21, 40)), (w, slice(72, 144)), (dy, slice(21, 40))):
        t[rows] = math.nan
        t[rows, ::3] = math.inf
    o = offsets(cuts)
    for bad, good in ((nv.linear_grouped(x, w, o), nv.linear_grouped(clean[0], clean[1], o)),
                      (nv.linear_grouped_backward(dy, x, w, o)[0],
                       nv.linear_grouped_backward(clean[2], clean[0], clean[1], o)[0])):
        assert torch.equal(bad[:21], good[:21]) and torch.equal(bad[40:], good[40:])
        assert not torch.isfinite(bad[21:40]).any()
    bad = nv.linear_grouped_backward(dy, x, w, o, bias_grad=True)
    good = nv.linear_grouped_backward(clean[2], clean[0], clean[1], o, bias_grad=True)
    for i, n in ((1, 72), (2, 1)):
        assert torch.equal(bad[i][:n], good[i][:n]) and torch.equal(bad[i][2 * n:], good[i][2 * n:])


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("M,N,K", [(1, 32, 8), (7, 96, 72), (64, 256, 256), (65, 288, 520), (130, 544, 64),
                                   (333, 1024, 264), (1000, 160, 136)])
def test_backward(nv, cuda_dev, act, M, N, K):
    for dtype in (torch.bfloat16, torch.float16):
        No = N // 2 if act == "swiglu" else N
        x, w, dy = make((M, K), dtype, 1), make((N, K), dtype, 2, K ** -0.5), make((M, No), dtype, 3)
        z = make((M, N), dtype, 4)
        got = nv.linear_backward(dy, x, w, preact=z if act != "none" else None, activation=act, bias_grad=True)
        nv.device_status()
        ref = R.backward64(dy, x, w, [0, M], z, act)
        for a, (r, e), n in zip(got, ref, ("dx", "dw", "db")):
            R.assert_close(a, r.reshape(a.shape), e.reshape(a.shape), n)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh", "swiglu"])
def test_gradient_of_the_epilogue_is_rounded_once(nv, cuda_dev, act):
    """The products of the backward pass take dZ = dY act'(Z) in the 16-bit type, rounded as the
    activation's gradient leaves it; the bias gradient sums it unrounded.  In fp16 a dZ past
    65504 is an infinity, and no dX that it enters is finite."""
    M, N, K = 70, 96, 72
    for dtype in (torch.bfloat16, torch.float16):
        No = N // 2 if act == "swiglu" else N
        x, w, dy = make((M, K), dtype, 1), make((N, K), dtype, 2), make((M, No), dtype, 3)
        z = make((M, N), dtype, 4)
        dz = torch.empty(M, N, dtype=dtype, device="cuda")
        s = torch.cuda.current_stream().cuda_stream

        def rounded(dy):
            assert nv.lib().nvfp4_activation_backward(dy.data_ptr(), z.data_ptr(), dz.data_ptr(), None, None, 1, M, N,
                                                      nv._lib.ACTIVATIONS[act], int(dtype == torch.float16), None, 0,
                                                      s) == 0
            return dz

        got = nv.linear_backward(dy, x, w, preact=z, activation=act)
        want = nv.linear_backward(rounded(dy), x, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for row, v in ((3, 4.0), (5, 1.5), (7, 2.4)):
        z[row], dy[row] = v, 60000.0
    past = R.dact64(dy.double(), z.double(), act).abs() >= 65520  # halfway to the next step of fp16
    assert torch.equal(rounded(dy).isinf(), past) and past.any() == (act != "relu")
    assert not nv.linear_backward(dy, x, w, preact=z, activation=act)[0][past.any(1)].isfinite().any()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
def test_backward_of_large_preactivations(nv, cuda_dev, act):
    """Pre-activations up to the largest bf16 value, whose square passes fp32, and infinities:
    the slope is 0 or 1 there."""
    v = torch.tensor([-math.inf, -3.38e38, -1e30, -6e19, -1e10, -300.0, -90.0, 90.0, 300.0, 1e10, 6e19, 1e30, 3.38e38,
                      math.inf, 0.0, 1.0], device="cuda").bfloat16()
    N = v.numel()
    x, w = make((4, 8), torch.bfloat16, 1), make((N, 8), torch.bfloat16, 2)
    dy, z = make((4, N), torch.bfloat16, 3), v.expand(4, N).contiguous()
    got = nv.linear_backward(dy, x, w, preact=z, activation=act, bias_grad=True)
    # infinities: the limits, which are the slopes at the largest values
    for a, (r, e), n in zip(got, R.backward64(dy, x, w, [0, 4], z.clamp(-3.38e38, 3.38e38), act), ("dx", "dw", "db")):
        R.assert_close(a, r.reshape(a.shape), e.reshape(a.shape), n)


@pytest.mark.parametrize("cuts", GROUPS, ids=lambda c: f"G{len(c) - 1}M{c[-1]}")
def test_backward_groups(nv, cuda_dev, cuts):
    for act, N, K, dtype in (("none", 72, 264, torch.bfloat16), ("swiglu", 288, 136, torch.bfloat16),
                             ("relu", 264, 72, torch.float16)):
        M, G, No = cuts[-1], len(cuts) - 1, N // 2 if act == "swiglu" else N
        x, w, dy = make((M, K), dtype, 1), make((G * N, K), dtype, 2, K ** -0.5), make((M, No), dtype, 3)
        z = make((M, N), dtype, 4)
        got = nv.linear_grouped_backward(dy, x, w, offsets(cuts), preact=z, activation=act, bias_grad=True)
        nv.device_status()
        for a, (r, e), n in zip(got, R.backward64(dy, x, w, cuts, z, act), ("dx", "dw", "db")):
            R.assert_close(a, r, e, n)


@pytest.mark.parametrize("M,cuts", [(5, None), (300, None), (300, [0, 100, 100, 290])])
def test_wanted_gradients_only(nv, cuda_dev, M, cuts):
    """Leaving out a gradient leaves the others' bits, and launches what is left."""
    G, N, K = 1 if cuts is None else len(cuts) - 1, 96, 136
    x, w, dy = make((M, K), torch.bfloat16, 1), make((G * N, K), torch.bfloat16, 2), make((M, N), torch.bfloat16, 3)
    z = make((M, N), torch.bfloat16, 4)

    def run(**wanted):
        n = nv.launch_count()
        if cuts is None:
            out = nv.linear_backward(dy, x, w, preact=z, activation="silu", **wanted)
        else:
            out = nv.linear_grouped_backward(dy, x, w, offsets(cuts), preact=z, activation="silu", **wanted)
        return out, nv.launch_count() - n

    (dx, dw, db), n = run(bias_grad=True)
    assert n == 4
    for want in ((1, 0, 1), (0, 1, 1), (0, 0, 1), (1, 0, 0), (0, 1, 0)):
        got, n = run(input_grad=bool(want[0]), weight_grad=bool(want[1]), bias_grad=bool(want[2]))
        assert n == 1 + sum(want)
        for a, b, on in zip(got, (dx, dw, db), want):
            assert (a is None) if not on else torch.equal(a, b)


@pytest.mark.parametrize("act", R.ACTS)
def test_gradient_against_differences(nv, cuda_dev, act):
    """<dL/dp, d> against (L(p + h d) - L(p - h d)) / 2h of the 64-bit forward pass, for
    L = <y, dy>.  The operator's gradients are off by a few roundings u of 16-bit values (a
    relative error of the inner product below 4u of the norms' product); the difference
    quotient is off by O(h^2)."""
    M, N, K, dtype = 24, 64, 40, torch.float16
    x, w, b = make((M, K), dtype, 1), make((N, K), dtype, 2, 0.3), make((N,), dtype, 3)
    dy = make((M, N // 2 if act == "swiglu" else N), dtype, 4)
    y, z = nv.linear(x, w, bias=b, activation=act, return_preact=True)
    grads = nv.linear_backward(dy, x, w, preact=z, activation=act, bias_grad=True)
    for i, p in enumerate((x, w, b)):
        d = make(p.shape, torch.float16, 10 + i).double()
        h = 1e-4

        def loss(s):
            q = [t.double() for t in (x, w, b)]
            q[i] = q[i] + s * d
            return (R.act64(q[0] @ q[1].t() + q[2], act) * dy.double()).sum()

        diff = ((loss(h) - loss(-h)) / (2 * h)).item()
        got = (grads[i].double() * d).sum().item()
        norm = (grads[i].double().norm() * d.norm()).item()
        if act == "relu":  # entries whose sign flips within h d do not matter at this h
            assert abs(got - diff) <= 8 * R.U[dtype] * norm
        else:
            assert abs(got - diff) <= 4 * R.U[dtype] * norm + 1e-6 * norm


def test_same_bits_every_time(nv, cuda_dev):
    cuts = [0, 100, 101, 400]
    x, w, dy = make((400, 328), torch.bfloat16, 1), make((3 * 320, 328), torch.bfloat16, 2), make((400, 320), torch.bfloat16, 3)
    z, o = make((400, 320), torch.bfloat16, 4), offsets(cuts)

    def once():
        return [nv.linear_grouped(x, w, o, activation="silu"), nv.linear(x[:3], w[:320]), nv.linear(x, w[:320]),
                *nv.linear_grouped_backward(dy, x, w, o, preact=z, activation="silu", bias_grad=True)]

    first = once()
    for _ in range(5):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_side_stream_and_graph(nv, cuda_dev):
    """The calls run on the current stream, and a captured graph follows inputs and offsets
    that change in place."""
    x, w = make((96, 128), torch.bfloat16, 1), make((4 * 128, 128), torch.bfloat16, 2)
    o = offsets([0, 10, 20, 60, 96])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        nv.linear_grouped(x, w, o)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = nv.linear_grouped(x, w, o)
    for cuts in ([0, 10, 20, 60, 96], [0, 0, 50, 50, 90]):
        o.copy_(offsets(cuts))
        x.copy_(make((96, 128), torch.bfloat16, cuts[2]))
        g.replay()
        torch.cuda.synchronize()
        R.assert_close(y, *R.forward64(x, w, cuts, None, "none", None)[:2])


def test_decreasing_offsets_stay_in_the_workspace(nv, cuda_dev):
    """Offsets that decrease are a mistake that only the device sees: they count more 64-row
    chunks than the workspace holds, and none past its end is read."""
    G, M, N = 64, 640, 64
    o = offsets([0, M] * (G // 2) + [0])
    size = nv.lib().nvfp4_activation_backward_workspace_size(G, M, N)
    ws = torch.full((4 * G * M // 64 * N,), math.nan, device="cuda")  # room for every chunk, NaN past `size`
    dy = torch.ones(M, N, dtype=torch.bfloat16, device="cuda")
    db = torch.empty(G, N, dtype=torch.bfloat16, device="cuda")
    assert size // 4 < G // 2 * M // 64 * N < ws.numel()
    assert nv.lib().nvfp4_activation_backward(dy.data_ptr(), None, None, db.data_ptr(), o.data_ptr(), G, M, N, 0, 0,
                                              ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    nv.device_status()
    assert (db[0] == M).all() and not db[1].any() and torch.isfinite(db).all()


def test_gradient_of_many_rows(nv, cuda_dev):
    """More 64-row chunks than a grid's second dimension has blocks."""
    M, N, K = 64 * 65535 + 70, 8, 8
    g = torch.Generator("cuda").manual_seed(1)
    x, dy, z = (torch.randn(M, s, device="cuda", generator=g).bfloat16() for s in (K, N, N))
    w = make((N, K), torch.bfloat16, 2)
    dx, dw, db = nv.linear_backward(dy, x, w, preact=z, activation="relu", bias_grad=True)
    nv.device_status()
    for got, (r, e), n in zip((dx, dw, db), R.backward64(dy, x, w, [0, M], z, "relu"), ("dx", "dw", "db")):
        R.assert_close(got, r.reshape(got.shape), e.reshape(got.shape), n)


def test_large_offsets(nv, cuda_dev):
    """An output of more than 2^31 elements: the last rows are where they belong."""
    M, N, K = 140_000, 16_384, 64
    x, w = make((M, K), torch.bfloat16, 1), make((N, K), torch.bfloat16, 2)
    y = nv.linear(x, w)
    nv.device_status()
    for a in (0, 131_072 - 8, M - 16):
        R.assert_close(y[a:a + 16], *R.forward64(x[a:a + 16], w, [0, 16], None, "none", None)[:2])


def test_out(nv, cuda_dev):
    """out is written in place; it may be the residual, and shares memory with no other input."""
    M, K = 300, 136
    wide = make((M, 2 * K), torch.bfloat16, 1)
    x, w, r = wide[:, :K], make((K, K), torch.bfloat16, 2), make((M, K), torch.bfloat16, 3)
    want = nv.linear(x, w, residual=r, activation="silu")
    out = torch.empty_like(r)
    assert nv.linear(x, w, residual=r, activation="silu", out=out) is not None and torch.equal(out, want)
    nv.linear(x, w, residual=r, activation="silu", out=r)
    assert torch.equal(r, want)
    xc, b = x.contiguous(), make((M * K + K,), torch.bfloat16, 4)
    big = make((M + 1, K), torch.bfloat16, 5)
    o = torch.zeros(M * K, dtype=torch.int32, device="cuda")
    for call, name in ((lambda: nv.linear(xc, w, out=xc), "x"), (lambda: nv.linear(big[1:], w, out=big[:M]), "x"),
                       (lambda: nv.linear(x, w, out=wide.view(-1)[M * K:].view(M, K)), "x"),
                       (lambda: nv.linear(x[:K], w, out=w), "w"),
                       (lambda: nv.linear(x, w, bias=b[8:8 + K], out=b[:M * K].view(M, K)), "bias"),
                       (lambda: nv.linear(x, w, residual=big[1:], out=big[:M]), "residual"),
                       (lambda: nv.linear_grouped(x, w, o[:2], out=o.view(torch.bfloat16)[:M * K].view(M, K)),
                        "m_offsets")):
        with pytest.raises(ValueError, match="share memory with " + name):
            call()


def test_refusals(nv, cuda_dev):
    """Arguments of the wrong shape, type or device raise ValueError; a pointer that is not
    16-byte aligned is the library's to refuse."""
    x, w = make((8, 64), torch.bfloat16, 1), make((128, 64), torch.bfloat16, 2)
    o = offsets([0, 4, 8])
    for bad in (lambda: nv.linear(x.float(), w), lambda: nv.linear(x, w.half()), lambda: nv.linear(x, w.cpu()),
                lambda: nv.linear(x[:, :60], w[:, :60].contiguous()), lambda: nv.linear(x, w[:, ::2]),
                lambda: nv.linear(x, w, bias=w[0]), lambda: nv.linear(x, w, residual=x),
                lambda: nv.linear(x, w, activation="tanh"), lambda: nv.linear(x, w[:120], activation="swiglu"),
                lambda: nv.linear(x, w, out=x), lambda: nv.linear(x.t(), w), lambda: nv.linear_grouped(x, w, None),
                lambda: nv.linear_grouped(x, w, o.long()), lambda: nv.linear_grouped(x, w, o[:1]),
                lambda: nv.linear_grouped(x, w[:127], o), lambda: nv.linear_backward(x, x, w),
                lambda: nv.linear_backward(make((8, 128), torch.bfloat16, 3), x, w, activation="relu")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(nv.NVFP4Error):
        nv.linear(torch.zeros(8 * 72 + 4, dtype=torch.bfloat16, device="cuda")[4:4 + 8 * 72].view(8, 72)[:, :64], w)
    with pytest.raises(TypeError):
        nv.linear(x)
