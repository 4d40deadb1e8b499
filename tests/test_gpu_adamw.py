"""aipt_adamw_* against the formula in fp64."""
import pytest
import torch

from ai_path_tracer_denoiser_amd import api
from tests.layer_util import F, context, generator, u, within

pytestmark = pytest.mark.gpu

B1, B2, EPS, LR = 0.9, 0.999, 1e-8, 1e-3
SETS = [[1], [256], [257, 3], [5, 0, 255, 1024, 1, 7000], [33] * 300, [70000, 2, 1]]


def tensors(gen, sizes, scale, dtype=torch.float32, offset=0):
    out = []
    for n in sizes:
        m = torch.full((n + offset,), 7.0, device="cuda", dtype=dtype)
        m[offset:] = (torch.randn(n, generator=gen, device="cuda") * scale).to(dtype)
        out.append(m[offset:])
    return out


def segments(sizes):
    at, out = 0, []
    for n in sizes:
        out.append(slice(at, at + n))
        at += -(-n // 256) * 256
    return out, at


def make_state(gen, sizes, bits, step):
    segs, total = segments(sizes)
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for s in segs:
        n = s.stop - s.start
        m[s], v[s] = torch.randn(n, generator=gen, device="cuda") * 1e-3, (torch.randn(n, generator=gen, device="cuda") * 2e-3).square() + 1e-9
    st = {"step": torch.full((1,), step, device="cuda", dtype=torch.int32)}
    if bits == 32:
        return {**st, "m": m, "v": v}
    for name, q in (("m", m), ("v", v.sqrt())):
        q = q.view(-1, 256)
        scale = q.abs().amax(1) / 448
        st[name] = (q / scale.clamp(min=1e-30)[:, None]).to(torch.float8_e4m3fn).view(-1)
        st[name + "_scale"] = scale
    return st


def values(st, bits):
    """m and v of a state in fp64."""
    if bits == 32:
        return st["m"].double(), st["v"].double()
    m, r = ((st[n].double().view(-1, 256) * st[n + "_scale"].double()[:, None]).view(-1) for n in ("m", "v"))
    return m, r.square()


def check_step(sizes, bits, gtype=torch.float32, ctype=None, decay=0.01, max_norm=None, step=0, seed=3, offset=0, scale=1e-2):
    gen = generator(sum(sizes) + len(sizes) + bits)
    p, g = tensors(gen, sizes, 0.1, offset=offset), tensors(gen, sizes, scale, gtype, offset)
    copies = None if ctype is None else [torch.full((n,), 9.0, device="cuda", dtype=ctype) for n in sizes]
    st = make_state(gen, sizes, bits, step)
    m0, v0 = values(st, bits)
    p0 = [q.double().clone() for q in p]
    plan = context().adamw(p, g, copies=copies, weight_decay=decay, state_bits=bits, state=st)
    plan.update(LR, B1, B2, EPS, max_norm, seed)
    t = step + 1
    assert int(st["step"]) == t
    # the norm: at most 256 terms a lane, then a tree and fp64: 2^-15 holds for every size here; half of it after the root
    norm = torch.sqrt(sum((q.double().square().sum() for q in g), torch.zeros((), device="cuda").double()))
    clip, ec = 1.0, 0.0
    if max_norm is not None:
        assert abs(float(plan.norm) - float(norm)) <= 2.0 ** -15 * float(norm)
        clip = min(1.0, max_norm / (float(norm) + 1e-6))
        ec = 2.0 ** -14
    decays = [decay] * len(sizes) if isinstance(decay, float) else decay
    segs, total = segments(sizes)
    m1, v1 = values(st, bits)
    for i, s in enumerate(segs):
        gi = g[i].double() * clip
        m, v = B1 * m0[s] + (1 - B1) * gi, B2 * v0[s] + (1 - B2) * gi.square()
        # each term is a few roundings from exact; the betas themselves are within F as fp32 numbers
        em = 6 * F * (m0[s].abs() + gi.abs()) + ec * gi.abs()
        ev = 6 * F * (v0[s] + gi.square()) + 2 * ec * (1 - B2) * gi.square()
        if bits == 32:
            within(m1[s], m, em + 1e-44, "m")
            within(v1[s], v, ev + 1e-44, "v")
        rate = LR / (1 - B1 ** t)
        den = v.sqrt() / (1 - B2 ** t) ** 0.5 + EPS
        step_ = rate * m / den
        eden = (ev / (2 * v.sqrt().clamp(min=1e-30))) / (1 - B2 ** t) ** 0.5
        ep = rate * em / den + step_.abs() * (eden / den + 16 * F) + 4 * F * p0[i].abs()
        want = p0[i] * (1 - LR * decays[i]) - step_
        within(p[i], want, ep, "p")
        if copies is not None:
            assert torch.equal(copies[i], p[i].to(ctype))
    if bits == 8:
        check_rounding(st, sizes, B1, m0, v0, g, clip, ec, seed, t)
    else:
        keep = torch.ones(total, dtype=torch.bool, device="cuda")
        for s in segs:
            keep[s] = False
        assert not m1[keep].any() and not v1[keep].any()


def uniform(total, seed, t):
    mask = 0xFFFFFFFF
    x = (torch.arange(total, device="cuda") ^ ((seed + t * 0x9E3779B1) & mask)) & mask
    for factor, shift in ((0x9E3779B1, 15), (0xBB67AE85, 13), (0x3C6EF373, 16)):
        x = (x * factor) & mask
        x = x ^ (x >> shift)
    return (x >> 8).double() * 2.0 ** -24


def check_rounding(st, sizes, b1, m0, v0, g, clip, ec, seed, t):
    segs, total = segments(sizes)
    gi = torch.zeros(total, device="cuda").double()
    for s, q in zip(segs, g):
        gi[s] = q.double() * clip
    m, r = b1 * m0 + (1 - b1) * gi, (B2 * v0 + (1 - B2) * gi.square()).sqrt()
    rel = 2.0 ** -18 + 2 * ec                                             # of a value, and so of a scale
    for name, q in (("m", m), ("v", r)):
        q = q.view(-1, 256)
        top = q.abs().amax(1)
        within(st[name + "_scale"], top / 448, rel * top / 448 + 1e-44, name + "_scale")
        x, code = q / (top / 448).clamp(min=1e-300)[:, None], st[name].double().view(-1, 256)
        assert bool(((code == 0) | (top > 0)[:, None]).all())
        x = x * (top > 0)[:, None]
        unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        near = x.abs() * 2 * rel + 1e-9
        if name == "m":                                                   # to nearest: within half a step (the neighbouring binade's, where x is next to it)
            # and what fp32 makes of beta1 m + (1 - beta1) g, which may cancel: its error is of the two terms' size (as for 32-bit state), not the sum's
            terms = ((6 * F + ec) * (m0.abs() + gi.abs())).view(-1, 256) / (top / 448).clamp(min=1e-300)[:, None]
            assert bool(((code - x).abs() <= unit / 2 + near + terms * (top > 0)[:, None]).all())
        else:
            up = torch.floor(x / unit + uniform(total, seed, t).view(-1, 256)) * unit
            want = torch.where((up == 0) & (x > 0), 2.0 ** -9, up).clamp(max=448)
            edge = (x / unit + uniform(total, seed, t).view(-1, 256))
            unsure = (edge - edge.round()).abs() <= near / unit + 2.0 ** -22       # the chance falls on a border of fp32's error
            # (a value next to a power of two, where the step changes, is no border: from below it is 16 steps but for an e, which only a chance below e
            # does not carry up, and from above 8 double steps)
            assert bool(((code == want) | unsure).all())
            assert float(unsure.double().mean()) < 0.02 or total <= 1024
            assert bool(((code - x).abs() <= unit + near).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SETS)
def test_sizes(sizes, bits):
    check_step(sizes, bits)
    check_step(sizes, bits, max_norm=0.05, step=900)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ctype", [None, torch.bfloat16, torch.float16])
def test_types(ctype, gtype, bits):
    check_step([300, 1, 4096, 77], bits, gtype, ctype, decay=[0.1, 0.0, 0.01, 0.5], step=10)
    check_step([300, 1, 4096, 77], bits, gtype, ctype, max_norm=1e6, offset=1, step=100000)      # unaligned tensors; nothing to clip


def test_large_and_many():
    check_step([3_000_001, 255, 1_500_000], 8, torch.bfloat16, torch.bfloat16)
    check_step([3_000_001, 255, 1_500_000], 32, max_norm=0.1)
    check_step(list(range(0, 260)), 8, max_norm=0.5)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_dead_blocks(bits):
    p, g = [torch.ones(600, device="cuda")], [torch.zeros(600, device="cuda")]
    plan = context().adamw(p, g, weight_decay=0.0, state_bits=bits)
    for _ in range(3):
        plan.update(LR, max_norm=1.0, seed=1)
    assert bool((p[0] == 1).all()) and int(plan.state()["step"]) == 3 and float(plan.norm) == 0
    assert not any(v.float().any() for k, v in plan.state().items() if k != "step")
    g[0][300] = 1.0                                                       # one live element in a block of zeros
    plan.update(LR, seed=1)
    assert float(p[0][300]) != 1 and int((p[0] != 1).sum()) == 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
def test_norm_that_is_not_finite_skips_the_step(bits, bad):
    gen = generator(20)
    p, g = tensors(gen, [700, 40], 1.0), tensors(gen, [700, 40], 1.0)
    plan = context().adamw(p, g, state_bits=bits)
    plan.update(LR, max_norm=1.0)
    before = [q.clone() for q in p] + [v.clone() for v in plan.state().values()]
    g[1][3] = bad
    plan.update(LR, max_norm=1.0)
    after = p + list(plan.state().values())
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, after))
    assert not torch.isfinite(plan.norm).all()
    g[1][3] = 0.5
    plan.update(LR, max_norm=1.0)
    assert int(plan.state()["step"]) == 2 and torch.isfinite(p[1]).all()


def test_eight_bit_root_follows_the_gradients_size():
    """Gradients grow tenfold: v moves by 0.1 % of the difference a step, far less than a step of e4m3.  By chance rounding its mean over many elements
    follows the exact average; rounding to nearest would leave it where it is."""
    n = 256 * 512
    p, g = [torch.zeros(n, device="cuda")], [torch.full((n,), 1e-3, device="cuda")]
    st = context().adamw(p, g, state_bits=8).state()
    st["v_scale"].fill_(1e-3 / 256)
    st["v"].copy_(torch.full((n,), 256.0, device="cuda").to(torch.float8_e4m3fn))     # root 1e-3
    st["m"].zero_()
    plan = context().adamw(p, g, state_bits=8, state=st)
    g[0].fill_(1.2e-3)
    for k in range(100):
        plan.update(1e-6, seed=11)
    v = values(st, 8)[1]
    want = 0.999 ** 100 * 1e-6 + (1 - 0.999 ** 100) * 1.44e-6
    # A root is within a step (6 %) of exact at each update, by chance: its square's mean gains at most the variance, a 0.0004 th a step at the rates here
    # (0.05 % of 6 % ...), 3 % of v in 100; the mean over 131072 elements scatters by less than 0.1 %
    assert abs(float(v.mean()) / want - 1) < 0.03
    assert float(v.mean()) > 1.02e-6                                       # it has moved


def test_runs_of_steps_and_state_handed_on():
    """Five steps, the plan renewed from its state in between, are five steps of one plan; state and copies on another stream's context too."""
    gen = generator(21)
    sizes = [1000, 17]
    for bits in (32, 8):
        p = tensors(gen, sizes, 0.1)
        q = [t.clone() for t in p]
        grads = [tensors(gen, sizes, 0.01) for _ in range(5)]
        g1, g2 = [t.clone() for t in grads[0]], [t.clone() for t in grads[0]]
        one, two = context().adamw(p, g1, state_bits=bits), context().adamw(q, g2, state_bits=bits)
        other = api.Context(0)
        for k in range(5):
            for a, b, c in zip(g1, g2, grads[k]):
                a.copy_(c), b.copy_(c)
            one.update(LR, max_norm=0.3, seed=k)
            two.update(LR, max_norm=0.3, seed=k)
            two = (other if k % 2 else context()).adamw(q, g2, state_bits=bits, state=two.state())
        assert all(torch.equal(a, b) for a, b in zip(p, q))
        assert all(torch.equal(a.view(torch.uint8), two.state()[k].view(torch.uint8)) for k, a in one.state().items())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count(bits):
    gen = generator(22)
    s = torch.cuda.Stream()
    ctx = api.Context(0, stream=s.cuda_stream)
    sizes = [33] * 130                                                    # two launches
    p, g = tensors(gen, sizes, 0.1), tensors(gen, sizes, 0.01)
    q, h = [t.clone() for t in p], [t.clone() for t in g]
    plan, eager = ctx.adamw(p, g, state_bits=bits), context().adamw(q, h, state_bits=bits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        plan.update(LR, max_norm=0.1, seed=5)
    for k in range(4):
        for a, b in zip(g, h):
            a.copy_(torch.randn(33, generator=gen, device="cuda") * 0.01)
            b.copy_(a)
        graph.replay()
        eager.update(LR, max_norm=0.1, seed=5)
        torch.cuda.synchronize()
        assert int(plan.state()["step"]) == k + 1
        assert all(torch.equal(a, b) for a, b in zip(p, q)), k
        assert all(torch.equal(a.view(torch.uint8), eager.state()[n].view(torch.uint8)) for n, a in plan.state().items())


def test_refusals():
    c = context()
    p, g = [torch.zeros(300, device="cuda")], [torch.zeros(300, device="cuda")]
    for bad, word in [(lambda: c.adamw(p, [g[0][:299]]), "grad 0"), (lambda: c.adamw(p, g, state_bits=16), "state_bits"), (lambda: c.adamw(p, g, weight_decay=[0.1, 0.2]), "weight_decay"),
                      (lambda: c.adamw([p[0].double()], g), "param 0"), (lambda: c.adamw(p, g, copies=[torch.zeros(300, device="cuda")]), "copies"),
                      (lambda: c.adamw(p, p), "overlaps"), (lambda: c.adamw(p + p, g + g), "overlaps"), (lambda: c.adamw([p[0][::2]], [g[0][::2]]), "contiguous"),
                      (lambda: c.adamw(p, g, state={"m": p[0]}), "state"), (lambda: c.adamw(p, g).update(LR, beta1=1.0), "beta1"),
                      (lambda: c.adamw(p, g).update(LR, max_norm=-1.0), "max_norm"), (lambda: c.adamw(p, g).update(float("nan")), "lr"), (lambda: c.adamw([], []).update(LR), "no elements")]:
        with pytest.raises(api.AiptError, match=word):
            bad()
    plan = c.adamw(p, g)
    g[0].data = torch.ones(300, device="cuda")
    with pytest.raises(api.AiptError, match="moved"):
        plan.update(LR)
    plan.bind(g)
    plan.update(LR)
    assert float(p[0][0]) != 0
    plan.close()
    with pytest.raises(api.AiptError, match="closed"):
        plan.update(LR)


def test_plan_made_while_the_streams_are_busy():
    """The table is written behind the workspace's zeros, and behind the steps of the plan before, whatever the streams are."""
    sizes = [70000, 3, 1025]
    ctx, gen = api.Context(0), generator(31)
    start, grads = tensors(gen, sizes, 0.1), [tensors(gen, sizes, 1e-2), tensors(gen, sizes, 1e-2)]

    def run(c, wait):
        p = [t.clone() for t in start]
        torch.cuda.synchronize()
        if wait:
            big = torch.zeros(1 << 28, device="cuda")
            for _ in range(20):
                big.add_(1.0)
        plan = c.adamw(p, grads[0], weight_decay=0.01)
        for k in range(4):
            if k == 2:
                plan.bind(grads[1])
            plan.update(LR)
        torch.cuda.synchronize()
        return p, int(plan.state()["step"])

    (a, s), (b, t) = run(ctx, True), run(context(), False)
    assert s == t == 4 and all(torch.equal(x, y) for x, y in zip(a, b))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    captured = api.Context(0, stream=side.cuda_stream)
    p = [t.clone() for t in start]
    plan = captured.adamw(p, grads[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        plan.update(LR)
        with pytest.raises(api.AiptError, match="before a capture"):
            plan.bind(grads[1])
    graph.replay()
    torch.cuda.synchronize()
    assert int(plan.state()["step"]) == 1
