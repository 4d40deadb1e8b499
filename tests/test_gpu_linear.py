"""aipt_linear / aipt_linear_backward against the formulas in fp64."""
import math

import pytest
import torch

from ai_path_tracer_denoiser_amd import api
from tests.layer_util import F, TYPES, context, empty_like_layout, generator, least, matrix, u, untouched, within

pytestmark = pytest.mark.gpu

ACTS = ["none", "leaky", "silu", "gelu"]
SLOPE = 0.1


def act(z, name):
    if name == "leaky":
        return torch.where(z > 0, z, SLOPE * z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z


def act_slope(z, name):
    if name == "leaky":
        return torch.where(z > 0, 1.0, SLOPE).to(z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def forward_reference(x, w, bias, residual, name):
    """y, z and their bounds.  z: K products in fp32 and the bias, (K + 1) F of the magnitudes.  The activations' slopes are at most 1.13, and
    evaluating one in fp32 (a handful of operations and expf / erff, each within 2 F) is within 16 F of its argument and result."""
    xd, wd = x.double(), w.double()
    z, s = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        z, s = z + bias.double(), s + bias.double().abs()
    ez = (x.shape[1] + 1) * F * s
    y = act(z, name)
    ey = 1.13 * ez + 16 * F * z.abs()
    if residual is not None:
        y = y + residual.double()
        ey = ey + F * y.abs()
    t = x.dtype
    return y, ey + u(t) * (y.abs() + ey) + least(t), z, ez + u(t) * (z.abs() + ez) + least(t)


def check_forward(x, w, bias, residual, name, y_layout="rows", pad=0, offset=0, keep=True, ctx=None):
    m, n, t = x.shape[0], w.shape[0], x.dtype
    y, ym = empty_like_layout(m, n, t, y_layout, pad, offset)
    z, zm = empty_like_layout(m, n, t, y_layout, pad, offset) if keep else (None, None)
    (ctx or context()).linear(x, w, y, bias=bias, residual=residual, preact=z, act=name, slope=SLOPE)
    yr, yb, zr, zb = forward_reference(x, w, bias, residual, name)
    within(y, yr, yb, "y")
    assert untouched(ym, y)
    if keep:
        within(z, zr, zb, "z")
        assert untouched(zm, z)
    return y


SIZES = [(1, 1, 1), (1, 64, 128), (3, 5, 7), (64, 64, 64), (65, 63, 33), (1, 300, 1000), (17, 101, 909), (130, 257, 129), (1000, 32, 64), (333, 43, 10), (256, 512, 384), (5, 2048, 96), (700, 3, 640)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward_sizes(m, n, k, dtype):
    gen = generator(m * 131 + n * 17 + k)
    x, w = matrix(gen, m, k, dtype), matrix(gen, n, k, dtype, scale=k ** -0.5)
    check_forward(x, w, matrix(gen, 1, n, dtype)[0], matrix(gen, m, n, dtype), ACTS[(m + n + k) % 4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_forward_activations(name, dtype):
    gen = generator(5)
    x, w = matrix(gen, 70, 48, dtype, scale=3), matrix(gen, 90, 48, dtype)       # arguments beyond +-30
    check_forward(x, w, None, None, name)
    check_forward(x, w, matrix(gen, 1, 90, dtype)[0], None, name, keep=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("xl,wl,yl", [(a, b, c) for a in ("rows", "planar") for b in ("rows", "planar") for c in ("rows", "planar")])
def test_forward_layouts(xl, wl, yl, dtype):
    for m, n, k, pad, offset in [(200, 136, 160, 0, 0), (200, 136, 160, 24, 8), (101, 57, 77, 3, 1)]:
        gen = generator(m + pad)
        x, w = matrix(gen, m, k, dtype, xl, pad=pad, offset=offset), matrix(gen, n, k, dtype, wl, scale=k ** -0.5, pad=pad, offset=offset)
        check_forward(x, w, matrix(gen, 1, n, dtype)[0], matrix(gen, m, n, dtype, "planar" if xl == "rows" else "rows", pad=pad), "silu", yl, pad, offset)


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_of_nothing(dtype):
    gen = generator(1)
    for m, n, k in [(0, 5, 4), (5, 0, 4), (0, 0, 0)]:
        context().linear(torch.empty(m, k, device="cuda", dtype=dtype), torch.empty(n, k, device="cuda", dtype=dtype), torch.empty(m, n, device="cuda", dtype=dtype))
    x, w = torch.empty(40, 0, device="cuda", dtype=dtype), torch.empty(30, 0, device="cuda", dtype=dtype)
    check_forward(x, w, matrix(gen, 1, 30, dtype)[0], matrix(gen, 40, 30, dtype), "gelu")        # no products: the bias
    check_forward(x, w, None, None, "none")


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_in_place_and_broadcast_inputs(dtype):
    gen = generator(2)
    for k in (96, 5000):             # (the second with its contraction split)
        x, w, r = matrix(gen, 60, k, dtype), matrix(gen, 80, k, dtype, scale=k ** -0.5), matrix(gen, 60, 80, dtype)
        y = r.clone()
        context().linear(x, w, y, residual=y, act="leaky", slope=SLOPE)
        yr, yb, _, _ = forward_reference(x, w, None, r, "leaky")
        within(y, yr, yb)
        check_forward(x[:1].expand(60, k), w, None, r[:1].expand(60, 80), "none")


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values_stay_in_their_rows(dtype):
    gen = generator(3)
    x, w = matrix(gen, 130, 200, dtype), matrix(gen, 70, 200, dtype)
    x[7, 3], x[64, 199], x[129, 0] = float("inf"), float("nan"), -float("inf")
    y = torch.empty(130, 70, device="cuda", dtype=dtype)
    context().linear(x, w, y)
    z = x.double() @ w.double().t()
    odd = torch.zeros(130, dtype=torch.bool, device="cuda")
    odd[[7, 64, 129]] = True
    assert torch.isfinite(y[~odd]).all() and torch.isnan(y[64]).all()
    assert torch.equal(y[7].double(), z[7]) and torch.equal(y[129].double(), z[129])             # infinities of the right signs


def backward_reference(dy, x, w, z, name):
    """dx, dw, dbias and their bounds.  dz: the slope within 16 F of its size (at most 1.13) and of 1, then rounded to the type; the products'
    sums of N, and of M, terms in fp32.  The bias' gradient adds unrounded dz."""
    t = dy.dtype
    d, xd, wd = dy.double(), x.double(), w.double()
    dz = d * act_slope(z.double(), name) if name != "none" else d
    e32 = 32 * F * d.abs() if name != "none" else torch.zeros_like(d)
    e = e32 + (u(t) * dz.abs() + least(t) if name != "none" else 0)
    big = dz.abs() + e
    m, n = d.shape
    def held(v, ev):
        return ev + u(t) * (v.abs() + ev) + least(t)
    dx, dw, db = dz @ wd, dz.t() @ xd, dz.sum(0)
    edx = e @ wd.abs() + n * F * (big @ wd.abs())
    edw = e.t() @ xd.abs() + m * F * (big.t() @ xd.abs())
    edb = e32.sum(0) + m * F * big.sum(0)
    return (dx, held(dx, edx)), (dw, held(dw, edw)), (db, held(db, edb))


def check_backward(dy, x, w, z, name, layout="rows", pad=0, offset=0, wanted=(True, True, True)):
    m, n, k, t = dy.shape[0], dy.shape[1], x.shape[1], dy.dtype
    dx, mx = empty_like_layout(m, k, t, layout, pad, offset)
    dw, mw = empty_like_layout(n, k, t, layout, pad, offset)
    db, mb = empty_like_layout(1, n, t, "rows", 0, offset)
    out = [v if f else None for v, f in zip((dx, dw, db[0]), wanted)]
    context().linear_backward(dy, x, w, preact=z, act=name, slope=SLOPE, dx=out[0], dw=out[1], dbias=out[2])
    for what, got, (want, bound), memory, view in zip(("dx", "dw", "dbias"), out, backward_reference(dy, x, w, z, name), (mx, mw, mb), (dx, dw, db)):
        if got is not None:
            within(got, want, bound, what)
            assert untouched(memory, view), what
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES + [(5000, 40, 30), (2, 3000, 9)])
def test_backward_sizes(m, n, k, dtype):
    gen = generator(m * 7 + n * 3 + k)
    name = ACTS[(m + n + k) % 4]
    check_backward(matrix(gen, m, n, dtype), matrix(gen, m, k, dtype), matrix(gen, n, k, dtype, scale=k ** -0.5), matrix(gen, m, n, dtype), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_backward_layouts(name, dtype):
    for m, n, k, pad, offset in [(200, 136, 160, 0, 0), (101, 57, 77, 3, 1), (96, 64, 128, 8, 8)]:
        for dl, xl, wl, ol in [("rows", "planar", "planar", "planar"), ("planar", "rows", "rows", "rows"), ("planar", "planar", "planar", "planar"), ("rows", "rows", "planar", "rows")]:
            gen = generator(m + pad)
            check_backward(matrix(gen, m, n, dtype, dl, pad=pad, offset=offset), matrix(gen, m, k, dtype, xl, pad=pad), matrix(gen, n, k, dtype, wl, pad=pad, offset=offset),
                           matrix(gen, m, n, dtype, xl, pad=pad), name, ol, pad, offset)


@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, False, False)])
def test_backward_of_some(wanted):
    gen = generator(4)
    for name in ("none", "gelu"):
        check_backward(matrix(gen, 150, 70, torch.float16), matrix(gen, 150, 40, torch.float16), matrix(gen, 70, 40, torch.float16), matrix(gen, 150, 70, torch.float16), name, wanted=wanted)
    dy = matrix(gen, 150, 70, torch.float32)
    db = torch.empty(70, device="cuda")
    context().linear_backward(dy, None, None, dbias=db)          # neither x nor w is needed for it
    within(db, dy.double().sum(0), 150 * F * dy.double().abs().sum(0) + u(torch.float32) * dy.double().sum(0).abs())


@pytest.mark.parametrize("dtype", TYPES)
def test_backward_of_nothing(dtype):
    x = torch.empty(0, 20, device="cuda", dtype=dtype)
    w = torch.ones(30, 20, device="cuda", dtype=dtype)
    dw, db = torch.ones(30, 20, device="cuda", dtype=dtype), torch.ones(30, device="cuda", dtype=dtype)
    dy = torch.empty(0, 30, device="cuda", dtype=dtype)
    context().linear_backward(dy, x, w, preact=dy.clone(), act="silu", dx=torch.empty_like(x), dw=dw, dbias=db)
    assert not dw.any() and not db.any()                         # sums of no rows
    x, w = torch.ones(20, 8, device="cuda", dtype=dtype), torch.empty(0, 8, device="cuda", dtype=dtype)
    dx = torch.ones_like(x)
    context().linear_backward(torch.empty(20, 0, device="cuda", dtype=dtype), x, w, dx=dx, dw=torch.empty_like(w), dbias=torch.empty(0, device="cuda", dtype=dtype))
    assert not dx.any()


def test_gradient_against_differences():
    """The loss sum(c * y) moves by the gradient times a small step: central differences of the fp64 formula, at the kernel's own gradients."""
    gen = generator(6)
    for name in ("leaky", "silu", "gelu"):
        x, w, b = matrix(gen, 9, 12, torch.float32), matrix(gen, 7, 12, torch.float32), matrix(gen, 1, 7, torch.float32)[0]
        c = matrix(gen, 9, 7, torch.float32)
        y, z = torch.empty(9, 7, device="cuda"), torch.empty(9, 7, device="cuda")
        context().linear(x, w, y, bias=b, preact=z, act=name, slope=SLOPE)
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        context().linear_backward(c, x, w, preact=z, act=name, slope=SLOPE, dx=dx, dw=dw, dbias=db)
        def loss(x, w, b):
            return (c.double() * act(x @ w.t() + b, name)).sum()
        args = [x.double(), w.double(), b.double()]
        for i, grad in enumerate((dx, dw, db)):
            step = torch.randn(args[i].shape, generator=gen, device="cuda").double()
            h = 1e-6                 # third derivatives times h^2 and the fp64 sums' error over h are both below 1e-8 here
            up, down = [a.clone() for a in args], [a.clone() for a in args]
            up[i] += h * step
            down[i] -= h * step
            want = float((loss(*up) - loss(*down)) / (2 * h))
            got = float((grad.double() * step).sum())
            assert abs(got - want) <= 1e-5 * float((grad.double() * step).abs().sum()) + 1e-7, (name, i)


def test_strides_beyond_32_bits():
    """Planes of 2^26 pixels: the last channel begins past 2^31 elements."""
    gen = generator(7)
    k, stride, m, n = 40, 1 << 26, 130, 50
    memory = torch.empty(k * stride, device="cuda", dtype=torch.float16)
    x = memory.view(k, stride)[:, stride - m:].t()
    x.copy_(torch.randn(m, k, generator=gen, device="cuda"))
    w = matrix(gen, n, k, torch.float16, scale=k ** -0.5)
    check_forward(x, w, None, None, "silu")
    y = memory.view(k, stride)[:, :m].t()                         # and as an output
    w2 = matrix(gen, k, n, torch.float16, scale=n ** -0.5)
    x2 = matrix(gen, m, n, torch.float16)
    context().linear(x2, w2, y)
    yr, yb, _, _ = forward_reference(x2, w2, None, None, "none")
    within(y, yr, yb)
    check_backward(matrix(gen, m, n, torch.float16), x, w, None, "none")


def test_own_stream_other_stream_and_same_bits():
    """A context with a stream of its own orders itself with torch's current stream; every stream gives the same bits."""
    gen = generator(8)
    own = api.Context(0)
    x, w = matrix(gen, 2000, 700, torch.bfloat16), matrix(gen, 300, 700, torch.bfloat16)
    want = torch.empty(2000, 300, device="cuda", dtype=torch.bfloat16)
    context().linear(x, w, want, act="gelu")
    side = torch.cuda.Stream()
    for _ in range(10):
        x2 = (x.float() * 2).to(torch.bfloat16)                  # queued on torch's stream just before
        y = torch.empty_like(want)
        own.linear(x2, w, y, act="gelu")
        context().linear(x, w, y, act="gelu")
        del x2
        assert torch.equal(y, want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2 = torch.empty_like(want)
            context().linear(x, w, y2, act="gelu")
            y2 = y2 * 1
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y2, want)


def test_captured_and_replayed():
    """Forward and backward in a graph, twice over with its own workspaces, replayed between eager calls on new inputs."""
    gen = generator(9)
    s = torch.cuda.Stream()
    ctx = api.Context(0, stream=s.cuda_stream)
    x, w = matrix(gen, 90, 4096, torch.bfloat16), matrix(gen, 70, 4096, torch.bfloat16, scale=1 / 64)     # split contractions: workspaces
    dy = matrix(gen, 90, 70, torch.bfloat16)
    def make():
        return {"y": torch.empty(90, 70, device="cuda", dtype=torch.bfloat16), "z": torch.empty(90, 70, device="cuda", dtype=torch.bfloat16),
                "dx": torch.empty_like(x), "dw": torch.empty_like(w), "db": torch.empty(70, device="cuda", dtype=torch.bfloat16)}
    def step(c, o):
        c.linear(x, w, o["y"], preact=o["z"], act="silu")
        c.linear_backward(dy, x, w, preact=o["z"], act="silu", dx=o["dx"], dw=o["dw"], dbias=o["db"])
    outs, graphs = [make(), make()], []
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step(ctx, outs[0])
    torch.cuda.synchronize()
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(ctx, o)
        graphs.append(g)
    eager = make()
    for i in range(4):
        x.copy_(matrix(gen, 90, 4096, torch.bfloat16))
        step(context(), eager)
        for o, g in zip(outs, graphs):
            for v in o.values():
                v.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            for name in o:
                assert torch.equal(o[name], eager[name]), (i, name)
    default = torch.cuda.CUDAGraph()
    with pytest.raises(api.AiptError, match="default stream"):
        with torch.cuda.graph(default):
            step(context(), eager)


# Rows whose numbers come close to 2^31: the last of what is added lies there.  Integers up to 256, which bf16 holds: exact.
@pytest.mark.parametrize("layout", ["rows", "planar"])
def test_backward_of_two_thousand_million_rows(layout):
    m, n = 2 ** 31 - 5000, 2
    shape = (m, n) if layout == "rows" else (n, m)
    turn = (lambda v: v) if layout == "rows" else (lambda v: v.t())
    dy, z, x = turn(torch.zeros(shape, device="cuda", dtype=torch.bfloat16)), turn(torch.full(shape, -1.0, device="cuda", dtype=torch.bfloat16)), torch.zeros(m, 1, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 1, 4097, 2 ** 20 + 3, 2 ** 30 - 1, 2 ** 30, 3 * 2 ** 29 + 77, m - 2 ** 21, m - 70000, m - 300, m - 65, m - 64, m - 9, m - 2, m - 1], device="cuda")
    dy[at, 0], dy[at, 1] = 2.0, 4.0
    x[at, 0] = (torch.arange(len(at), device="cuda") % 5 + 1).to(torch.bfloat16)
    dw, db = torch.full((n, 1), 9.0, device="cuda", dtype=torch.bfloat16), torch.full((n,), 9.0, device="cuda", dtype=torch.bfloat16)
    context().linear_backward(dy, x, None, preact=z, act="leaky", slope=0.5, dw=dw, dbias=db)
    total = float(x[at, 0].sum())
    assert dw.flatten().tolist() == [total, 2 * total] and db.tolist() == [float(len(at)), 2.0 * len(at)]


# Rows that begin at any element, their last ones short of a tile, a wave or eight elements: what lies between and behind them stays as it was.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [70, 20000])
@pytest.mark.parametrize("n", [7, 8, 9, 31, 33, 39, 41, 57, 63, 65, 71, 73, 127, 129, 143, 303])
def test_rows_that_begin_anywhere(n, m, dtype):
    gen = generator(n * 7 + m)
    k = 64
    x, w, b, r = matrix(gen, m, k, dtype), matrix(gen, n, k, dtype, scale=k ** -0.5), matrix(gen, 1, n, dtype)[0], matrix(gen, m, n, dtype, pad=1, offset=1)
    check_forward(x, w, b, r, ACTS[n % 4], pad=n % 3, offset=1)
    y = r.clone()
    context().linear(x, w, y, bias=b, residual=y, act="gelu")
    yr, yb, _, _ = forward_reference(x, w, b, r, "gelu")
    within(y, yr, yb)
    check_backward(*(matrix(gen, m, c, dtype) for c in (k, n)), matrix(gen, k, n, dtype, scale=n ** -0.5), matrix(gen, m, k, dtype), "silu", pad=n % 2, offset=1)
