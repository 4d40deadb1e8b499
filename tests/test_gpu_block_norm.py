"""aipt_block_norm / aipt_block_norm_backward against the formulas in fp64."""
import pytest
import torch

from ai_path_tracer_denoiser_amd import api
from tests.layer_util import F, TYPES, context, empty_like_layout, generator, least, matrix, u, untouched, within

pytestmark = pytest.mark.gpu

EPS = 1e-5
# Sums over a row: a lane adds at most 32 terms, then 6 exchanges and up to 16 waves: fewer than 64 roundings.  With the few roundings of a
# term itself, 2^-18 = 64 F of the terms' magnitudes covers every row sum; 16 F every chain of elementwise operations.
R, E = 2.0 ** -18, 16 * F


def parts(v, kind):
    """hat, mean, rstd of v in fp64, and a bound of what fp32 makes of hat, given the error `ev` of v."""
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = ((v - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
    return (v - mean) * rstd, mean, rstd


def hat_bound(v, ev, hat, rstd, kind):
    """Error of (v - mean) rstd: of v, of its mean, and the relative error of rstd -- half that of the mean square, which the error of the
    terms moves by 2 mean(|hat| e) rstd and its sum by R."""
    ec = ev + F * v.abs()
    if kind == "layer":
        ec = ec + ev.mean(1, keepdim=True) + R * v.abs().mean(1, keepdim=True)
    return rstd * ec + hat.abs() * (rstd * (hat.abs() * ec).mean(1, keepdim=True) + R + E), rstd * (rstd * (hat.abs() * ec).mean(1, keepdim=True) + R + E)


def vectors(gen, c, dtype, kind, groups):
    d = {"gate": matrix(gen, groups, c, dtype), "scale": 1 + 0.3 * matrix(gen, 1, c, dtype)[0], "post_weight": 1 + 0.3 * matrix(gen, 1, c, dtype)[0],
         "pre_weight": 1 + 0.3 * matrix(gen, 1, c, dtype)[0]}
    if kind == "layer":
        d.update(post_bias=0.2 * matrix(gen, 1, c, dtype)[0], pre_bias=0.2 * matrix(gen, 1, c, dtype)[0])
    return d


def f64(v, c):
    return {k: (v[k].double() if v.get(k) is not None else default) for k, default in
            (("gate", None), ("scale", torch.ones(c, device="cuda").double()), ("post_weight", torch.ones(c, device="cuda").double()), ("post_bias", torch.zeros(c, device="cuda").double()),
             ("pre_weight", torch.ones(c, device="cuda").double()), ("pre_bias", torch.zeros(c, device="cuda").double()))}


def check_forward(y, x, v, kind, z=True, stats=True, pad=0, offset=0, in_place=False):
    (m, c), t = x.shape, x.dtype
    xr = x.double()
    if in_place:
        h, hm = x, None
    else:
        h, hm = empty_like_layout(m, c, t, "rows", pad, offset)
    zt, zm = empty_like_layout(m, c, t, "rows", pad, offset) if z else (None, None)
    st = torch.full((m, 4), 5.0, device="cuda") if stats else None
    context().block_norm(y, x, h, zt, kind=kind, eps=EPS, stats=st, **v)
    f = f64(v, c)
    e = torch.zeros_like(xr)
    hr = xr
    if y is not None:
        yr = y.double()
        hat, my, ry = parts(yr, kind)
        eh, er = hat_bound(yr, torch.zeros_like(yr), hat, ry, kind)
        gate = f["gate"].repeat_interleave(m // f["gate"].shape[0], 0) if f["gate"] is not None else torch.ones_like(yr)
        k = f["scale"] * gate
        uu = hat * f["post_weight"] + f["post_bias"]
        hr = xr + k * uu
        e = k.abs() * (f["post_weight"].abs() * eh + E * ((hat * f["post_weight"]).abs() + f["post_bias"].abs())) + E * hr.abs()
        if stats:
            within(st[:, 1:2], ry, er, "rstd of y")
            within(st[:, 0:1], my, R * yr.abs().mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(my), "mean of y")
    within(h, hr, e + u(t) * (hr.abs() + e) + least(t), "h")
    assert hm is None or untouched(hm, h)
    if z:
        hat, mh, rh = parts(hr, kind)
        eh, er = hat_bound(hr, e, hat, rh, kind)
        zr = hat * f["pre_weight"] + f["pre_bias"]
        ez = f["pre_weight"].abs() * eh + E * ((hat * f["pre_weight"]).abs() + f["pre_bias"].abs())
        within(zt, zr, ez + u(t) * (zr.abs() + ez) + least(t), "z")
        assert untouched(zm, zt)
        if stats:
            within(st[:, 3:4], rh, er, "rstd of h")


WIDTHS = [1, 2, 3, 8, 43, 57, 64, 101, 128, 200, 512, 513, 700, 1024, 2040, 2047, 4096, 5000, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", WIDTHS)
def test_forward_widths(c, kind, dtype):
    gen = generator(c)
    m = 12 if c > 4000 else 36
    check_forward(matrix(gen, m, c, dtype, scale=2) + 0.5, matrix(gen, m, c, dtype), vectors(gen, c, dtype, kind, 3), kind)


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_parts_layouts_and_rows(dtype):
    gen = generator(11)
    for m, c, pad, offset in [(1, 64, 0, 0), (2, 300, 5, 3), (501, 96, 8, 8), (64, 96, 1, 0), (3000, 17, 0, 1)]:
        for kind in ("rms", "layer"):
            x, y = matrix(gen, m, c, dtype, pad=pad, offset=offset), matrix(gen, m, c, dtype, pad=pad)
            full = vectors(gen, c, dtype, kind, m)                        # a gate for every element
            check_forward(y, x, full, kind, pad=pad, offset=offset)
            check_forward(y, x, {}, kind, pad=pad)
            check_forward(y, x, {"gate": full["gate"][:1]}, kind, stats=False)
            check_forward(y, x, {k: full[k] for k in ("scale", "post_weight")}, kind, z=False)
            check_forward(None, x, {k: full[k] for k in ("pre_weight", "pre_bias") if k in full}, kind)
            check_forward(y, x, full, kind, in_place=True)
    context().block_norm(torch.empty(0, 8, device="cuda", dtype=dtype), torch.empty(0, 8, device="cuda", dtype=dtype), torch.empty(0, 8, device="cuda", dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_and_special_values(dtype):
    gen = generator(12)
    x, y = torch.zeros(6, 80, device="cuda", dtype=dtype), torch.zeros(6, 80, device="cuda", dtype=dtype)
    check_forward(y, x, {}, "rms")
    check_forward(y + 3, x, {}, "layer")                                  # a constant row: variance 0
    x, y = matrix(gen, 8, 80, dtype), matrix(gen, 8, 80, dtype)
    y[3, 5] = float("nan")
    y[5, 79] = float("inf")
    h, z = torch.empty_like(x), torch.empty_like(x)
    context().block_norm(y, x, h, z)
    keep = [i for i in range(8) if i not in (3, 5)]
    assert torch.isfinite(h[keep]).all() and torch.isfinite(z[keep]).all() and torch.isnan(z[3]).all()
    if dtype != torch.float16:                                            # squares up to 1e36 in bf16 / fp32: no overflow where the result has none
        check_forward(matrix(gen, 4, 64, dtype, scale=1e15), matrix(gen, 4, 64, dtype), {}, "rms")


def backward_reference(dh, dz, y, h, st, v, kind, m, c):
    """Results and bounds, from the stored statistics."""
    f = f64(v, c)
    d = lambda q: q.double() if q is not None else None
    dh, dz, y, h, st = d(dh), d(dz), d(y), d(h), st.double()
    out = {}
    zero = torch.zeros(m, c, device="cuda").double()
    t, et = (dh.clone(), zero.clone()) if dh is not None else (zero.clone(), zero.clone())

    def through(g, eg, hat, eh, rstd):
        """norm'(g), and its bound: of g, of hat, of the two row sums."""
        mean = g.mean(1, keepdim=True) if kind == "layer" else 0
        dot = (g * hat).mean(1, keepdim=True)
        e = eg + hat.abs() * (eg * hat.abs() + g.abs() * eh).mean(1, keepdim=True) + eh * dot.abs() + R * (hat.abs() * (g * hat).abs().mean(1, keepdim=True))
        if kind == "layer":
            e = e + eg.mean(1, keepdim=True) + R * g.abs().mean(1, keepdim=True)
        return rstd * (g - mean - hat * dot), rstd * (e + E * (g.abs() + (mean.abs() if kind == "layer" else 0) + (hat * dot).abs()))
    if dz is not None:
        hat = (h - st[:, 2:3]) * st[:, 3:4]
        eh = E * (h.abs() + st[:, 2:3].abs()) * st[:, 3:4]
        g = dz * f["pre_weight"]
        q, eq = through(g, E * g.abs(), hat, eh, st[:, 3:4])
        t, et = t + q, eq + E * (t.abs() + q.abs())
        out["dpre_weight"], out["dpre_bias"] = ((dz * hat).sum(0), (dz.abs() * eh + (m + 8) * F * (dz * hat).abs()).sum(0)), (dz.sum(0), m * F * dz.abs().sum(0))
    out["dx"] = (t, et)
    if y is not None:
        gate = f["gate"].repeat_interleave(m // f["gate"].shape[0], 0) if f["gate"] is not None else torch.ones_like(t)
        hat = (y - st[:, 0:1]) * st[:, 1:2]
        eh = E * (y.abs() + st[:, 0:1].abs()) * st[:, 1:2]
        uu = hat * f["post_weight"] + f["post_bias"]
        eu = f["post_weight"].abs() * eh + E * ((hat * f["post_weight"]).abs() + f["post_bias"].abs())
        k = gate * f["scale"]
        du, edu = t * k, et * k.abs() + E * (t * k).abs()
        g = du * f["post_weight"]
        out["dy"] = through(g, edu * f["post_weight"].abs() + E * g.abs(), hat, eh, st[:, 1:2])
        def column(terms, eterms, groups=1, times=1.0, loose=None):
            n = m // groups
            size = (terms.abs() if loose is None else loose).view(groups, n, c).sum(1)
            e = eterms.view(groups, n, c).sum(1) + (n + 24) * F * size
            s = terms.view(groups, n, c).sum(1)
            return (s * times, e * (times.abs() if torch.is_tensor(times) else times))
        sq = lambda p: (p[0][0], p[1][0])
        # scale's gradient is put together from the sums with and without the weight: their magnitudes count
        loose = (t * gate).abs() * ((hat * f["post_weight"]).abs() + f["post_bias"].abs())
        out["dscale"] = sq(column(t * gate * uu, gate.abs() * (et * uu.abs() + t.abs() * eu), loose=loose))
        groups = f["gate"].shape[0] if f["gate"] is not None else 1
        loose = t.abs() * ((hat * f["post_weight"]).abs() + f["post_bias"].abs())
        out["dgate"] = column(t * uu, et * uu.abs() + t.abs() * eu, groups, f["scale"], loose)
        out["dpost_weight"] = sq(column(t * gate * hat, gate.abs() * (et * hat.abs() + t.abs() * eh), 1, f["scale"]))
        out["dpost_bias"] = sq(column(t * gate, gate.abs() * et, 1, f["scale"]))
    return out


def check_backward(dh, dz, y, h, v, kind, pad=0, offset=0, skip=(), in_place=False):
    like = dh if dh is not None else dz
    (m, c), t = like.shape, like.dtype
    st = torch.zeros(m, 4, device="cuda")
    for i, q in ((0, y), (2, h)):
        if q is not None:
            _, mean, rstd = parts(q.double(), kind)
            st[:, i], st[:, i + 1] = mean[:, 0].float(), rstd[:, 0].float()
    want = backward_reference(dh, dz, y, h, st, v, kind, m, c)
    names = [n for n in want if n not in skip and not (kind == "rms" and "bias" in n) and not (n == "dgate" and v.get("gate") is None)]
    outs, memory = {}, {}
    for n in names:
        shape = (m, c) if n in ("dx", "dy") else tuple(want[n][0].shape) if n == "dgate" else (1, c)
        if n == "dx" and in_place:
            outs[n] = dh
            continue
        o, memory[n] = empty_like_layout(*shape, t, "rows", pad if n in ("dx", "dy") else 0, offset if n in ("dx", "dy") else 0)
        outs[n] = o if n in ("dx", "dy", "dgate") else o[0]
    fwd = {k: v.get(k) for k in ("gate", "scale", "post_weight", "post_bias", "pre_weight") if not (k == "pre_weight" and dz is None)}
    context().block_norm_backward(dh, dz, y, h, st, kind=kind, **fwd, **outs)
    for n in names:
        w, e = want[n]
        within(outs[n], w, e + u(t) * (w.abs() + e) + least(t), n)
        if n in memory and n in ("dx", "dy"):
            assert untouched(memory[n], outs[n]), n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", WIDTHS)
def test_backward_widths(c, kind, dtype):
    gen = generator(c + 1)
    m = 12 if c > 4000 else 60
    q = [matrix(gen, m, c, dtype) for _ in range(4)]
    check_backward(q[0], q[1], q[2] + 0.4, q[3] + 0.2, vectors(gen, c, dtype, kind, 3), kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,c,groups", [(1, 40, 1), (40, 24, 40), (999, 30, 3), (20000, 57, 1), (20000, 8, 4), (12000, 5, 6000), (9000, 16, 9000), (8192, 1024, 2), (5000, 520, 2500), (6000, 257, 6)])
def test_backward_rows_and_gates(m, c, groups, dtype):
    gen = generator(m + c)
    kind = "layer" if c % 2 else "rms"
    q = [matrix(gen, m, c, dtype) for _ in range(4)]
    check_backward(q[0], q[1], q[2], q[3], vectors(gen, c, dtype, kind, groups), kind)


@pytest.mark.parametrize("dtype", TYPES)
def test_backward_parts_and_layouts(dtype):
    gen = generator(13)
    for m, c, pad, offset in [(50, 64, 0, 0), (51, 72, 8, 8), (33, 70, 3, 1)]:
        for kind in ("rms", "layer"):
            q = [matrix(gen, m, c, dtype, pad=pad, offset=offset) for _ in range(4)]
            v = vectors(gen, c, dtype, kind, 1)
            check_backward(*q, v, kind, pad, offset)
            check_backward(None, *q[1:], v, kind)
            check_backward(q[0], None, q[2], None, v, kind)                                   # no norm before a next block
            check_backward(q[0], q[1], None, q[3], {"pre_weight": v["pre_weight"]}, kind)     # no block
            check_backward(*q, {}, kind)
            check_backward(*q, v, kind, skip=("dgate", "dscale", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"))
            check_backward(*q, v, kind, skip=("dx", "dscale", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"))
            check_backward(*q, v, kind, skip=("dy", "dgate"))
            check_backward(*q, v, kind, in_place=True)


def test_backward_of_no_rows():
    e = torch.empty(0, 24, device="cuda")
    for groups in (1, 3):
        o = {n: torch.ones(24, device="cuda") for n in ("dscale", "dpost_weight", "dpre_weight")}
        dg = torch.ones(groups, 24, device="cuda")
        context().block_norm_backward(e, e.clone(), e.clone(), e.clone(), torch.empty(0, 4, device="cuda"), gate=torch.ones(groups, 24, device="cuda"), dx=e.clone(), dy=e.clone(), dgate=dg, **o)
        assert not dg.any() and not any(v.any() for v in o.values())


def test_gradient_against_differences():
    gen = generator(14)
    for kind in ("rms", "layer"):
        m, c, groups = 6, 10, 2
        v = {k: q.float() for k, q in vectors(gen, c, torch.float32, kind, groups).items()}
        x, y, ch, cz = (matrix(gen, m, c, torch.float32) for _ in range(4))
        h, z, st = torch.empty_like(x), torch.empty_like(x), torch.empty(m, 4, device="cuda")
        context().block_norm(y, x, h, z, kind=kind, eps=EPS, stats=st, **v)
        names = ["gate", "scale", "post_weight", "pre_weight"] + (["post_bias", "pre_bias"] if kind == "layer" else [])
        grads = {"d" + n: torch.empty_like(v[n]) for n in names}
        dx, dy = torch.empty_like(x), torch.empty_like(x)
        context().block_norm_backward(ch, cz, y, h, st, kind=kind, **{n: v.get(n) for n in ("gate", "scale", "post_weight", "post_bias", "pre_weight")}, dx=dx, dy=dy, **grads)

        def loss(a):
            hat, _, _ = parts(a["y"], kind)
            hh = a["x"] + a["scale"] * a["gate"].repeat_interleave(m // groups, 0) * (hat * a["post_weight"] + a.get("post_bias", 0))
            zz = parts(hh, kind)[0] * a["pre_weight"] + a.get("pre_bias", 0)
            return (ch.double() * hh).sum() + (cz.double() * zz).sum()
        args = {k: q.double() for k, q in {**v, "x": x, "y": y}.items()}
        for n, grad in [("x", dx), ("y", dy)] + [(n, grads["d" + n]) for n in names]:
            step = torch.randn(args[n].shape, generator=gen, device="cuda").double()
            s = 1e-6
            want = float((loss({**args, n: args[n] + s * step}) - loss({**args, n: args[n] - s * step})) / (2 * s))
            got = float((grad.double() * step).sum())
            assert abs(got - want) <= 3e-5 * float((grad.double() * step).abs().sum()) + 1e-6, (kind, n, got, want)


def test_same_bits_and_captured():
    gen = generator(15)
    s = torch.cuda.Stream()
    ctx = api.Context(0, stream=s.cuda_stream)
    m, c = 3000, 96
    x, y, dh, dz = (matrix(gen, m, c, torch.bfloat16) for _ in range(4))
    v = vectors(gen, c, torch.bfloat16, "layer", 3)
    def make():
        return {n: torch.empty_like(x) for n in ("h", "z", "dx", "dy")} | {"st": torch.empty(m, 4, device="cuda")} | {"d" + n: torch.empty_like(q) for n, q in v.items()}
    def step(k, o):
        k.block_norm(y, x, o["h"], o["z"], kind="layer", stats=o["st"], **v)
        k.block_norm_backward(dh, dz, y, o["h"], o["st"], kind="layer", **{n: v[n] for n in v if n != "pre_bias"}, dx=o["dx"], dy=o["dy"], **{"d" + n: o["d" + n] for n in v})
    captured, eager = make(), make()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step(ctx, captured)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(ctx, captured)
    for _ in range(4):
        y.copy_(matrix(gen, m, c, torch.bfloat16))
        step(context(), eager)
        for q in captured.values():
            q.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(eager[n], captured[n]), n


# A workgroup goes through several rows, their gates change on the way, and each way of reading a row (16 bytes, two elements, one) is taken.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,c,groups", [(150000, 24, 3), (150000, 24, 75000), (40000, 57, 5), (40000, 38, 40000), (9000, 600, 9), (9000, 602, 2), (9000, 601, 9000), (3600, 1500, 3), (3600, 1501, 1), (3600, 1502, 1800),
                                        (1200, 4500, 400), (1200, 4502, 3), (1200, 4501, 3), (800, 6100, 2), (800, 6801, 4), (600, 9000, 6), (600, 9001, 1), (600, 9002, 300)])
def test_several_rows_a_workgroup(m, c, groups, dtype):
    gen = generator(m + c)
    for kind, in_place in (("layer", False), ("rms", True)):
        check_forward(matrix(gen, m, c, dtype), matrix(gen, m, c, dtype), vectors(gen, c, dtype, kind, groups), kind, in_place=in_place)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", [16, 30, 32, 60, 66, 130, 258, 514, 998, 1000, 1026, 2049, 2050, 4097, 4098, 6146, 6150, 7001])
def test_backward_more_widths(c, kind, dtype):
    gen = generator(c + 2)
    m = 2700 if c < 1000 else 1500
    check_backward(*(matrix(gen, m, c, dtype) for _ in range(4)), vectors(gen, c, dtype, kind, 3), kind)
