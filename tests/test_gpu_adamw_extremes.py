"""AdamW where the numbers are extreme: gradients and states at the ends of fp32, and what is none."""
import pytest
import torch

from tests.layer_util import F, context, generator, within
from tests.test_gpu_adamw import LR, make_state, segments, tensors, values

pytestmark = pytest.mark.gpu

SIZES = [600, 7]                                         # blocks of 256, 256, 88 and 7 elements


@pytest.mark.parametrize("bad", [float("nan"), -float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
def test_a_gradient_that_is_no_number_spoils_its_blocks_state_and_no_other(gtype, bad):
    """8-bit state, no clipping: all of the block's m and v, none of another's; its element alone with 32 bits."""
    for bits in (8, 32):
        plans = []
        for spoil in (False, True):
            gen = generator(50)
            p, g, st = tensors(gen, SIZES, 0.1), tensors(gen, SIZES, 0.01, gtype), make_state(gen, SIZES, bits, 5)
            if spoil:
                g[0][300] = bad
            plan = context().adamw(p, g, state_bits=bits, state=st)
            plan.update(LR, seed=3)
            plans.append((p, st))
        (p, good), (q, odd) = plans
        spoilt = torch.zeros(1024, dtype=torch.bool, device="cuda")
        spoilt[256:512] = True
        if bits == 32:
            spoilt[:] = False
            spoilt[300] = True
        for a, b in zip(values(good, bits), values(odd, bits)):
            assert not torch.isfinite(b[spoilt]).any() and torch.equal(a[~spoilt], b[~spoilt])
        assert torch.equal(p[1], q[1]) and not torch.isfinite(q[0][300])
        plan.update(LR, seed=4)                          # a step later it is still seen
        assert not any(torch.isfinite(v[spoilt][:1]).any() for v in values(odd, bits)) and torch.isfinite(q[1]).all()


def test_an_eps_of_nothing_and_subnormal_second_moments():
    """32-bit state: the step lr m / sqrt(v) of a v below 2^-126 is what the formula says."""
    n = 512
    v0 = torch.logspace(-44, -30, n, dtype=torch.float64, device="cuda").float()
    m0 = torch.full((n,), 1e-22, device="cuda")
    p, g = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
    st = {"m": m0.clone(), "v": v0.clone(), "step": torch.full((1,), 1000, device="cuda", dtype=torch.int32)}
    plan = context().adamw(p, g, weight_decay=0.0, state=st)
    plan.update(LR, eps=0.0)
    m, v = 0.9 * m0.double(), 0.999 * v0.double()
    want = -LR / (1 - 0.9 ** 1001) * m / (v / (1 - 0.999 ** 1001)).sqrt()
    # v = beta2 v0: beta2 is an fp32 number, within F of 0.999, and the product is rounded, by F or by half of 2^-149: together (1 + F)(1 + F) - 1, 2 F of it
    # to first order, and 2^-150.  Its root feels half of that; beside it 8 roundings and the ulp each of root and reciprocal
    ev = (2.0 ** -150 + 2 * F * v) / v
    within(st["v"], v, ev * v, "v")
    within(p[0], want, want.abs() * (ev / 2 / (1 - ev) + 12 * F), "p")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e20, 1e-30])
def test_the_norm_of_gradients_whose_squares_are_no_floats(size, gtype, bits):
    """1e20, whose square is beyond fp32's largest: clipped like any other; 1e-30, whose square is below its least: the norm is not zero."""
    gen = generator(51)
    p, g = tensors(gen, SIZES, 0.0), tensors(gen, SIZES, size, gtype)
    plan = context().adamw(p, g, weight_decay=0.0, state_bits=bits)
    plan.update(LR, max_norm=0.5)
    norm = torch.cat([t.double() for t in g]).square().sum().sqrt()
    # fp64 sums and root (errors of 2^-44 at these sizes), one rounding to fp32
    assert abs(float(plan.norm) - float(norm)) <= 1.01 * F * float(norm)
    assert int(plan.state()["step"]) == 1
    clipped = [t.double() * min(1.0, 0.5 / (float(norm) + 1e-6)) for t in g]
    # the first step of a plan is lr g / (|g| + eps), eps and |g| taken by a root each: 24 F of its terms, a factor's 4 F among them.
    # Below 1e-18 the square is no normal number and the step g / eps: within v's root of nothing, which is |g| at most (and eps is 1e12 of them)
    for a, c in zip(p, clipped):
        want = -LR * c / (c.abs() + 1e-8)
        within(a, want, want.abs() * 24 * F + (LR * c.abs() / 1e-8 if size < 1 else 0) + 1e-44, "p")
