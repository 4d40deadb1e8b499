"""The activations of aipt_linear and their slopes over the whole range, relative to their own size: what is small is right in its digits too."""
import math

import pytest
import torch

from tests.layer_util import F, TYPES, context, least, u, within
from tests.test_gpu_linear import act, act_slope

pytestmark = pytest.mark.gpu


def arguments(dtype, low, high):
    z = torch.cat([torch.linspace(low, high, 40001, device="cuda"), -torch.logspace(-30, 0, 500, device="cuda"), torch.logspace(-30, 0, 500, device="cuda"), torch.zeros(1, device="cuda")])
    return z.to(dtype)[:, None]


def normal(z):
    """phi and Phi in fp64, both to their last digits."""
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-z / math.sqrt(2))


def results(z, name):
    """act and slope of z by the kernels: a product with 1 is exact, and so is the one that the gradient takes."""
    y, one, dx = torch.empty(z.shape[0], 3, device="cuda", dtype=z.dtype), torch.ones(3, 1, device="cuda", dtype=z.dtype), torch.empty_like(z)
    context().linear(z, one, y, act=name)
    bits = y.view(torch.int32 if y.element_size() == 4 else torch.int16)
    assert torch.equal(bits[:, 0], bits[:, 1]) and torch.equal(bits[:, 0], bits[:, 2])
    context().linear_backward(torch.ones_like(z), z, one[:1], preact=z, act=name, dx=dx)
    return y[:, 0], dx[:, 0]


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_to_the_end_of_its_tail(dtype):
    z = arguments(dtype, -13, 13)
    y, d = results(z, "gelu")
    z = z[:, 0].double()
    pdf, cdf = normal(z)
    # Phi.  Floats: the fit 0.2 F; the reciprocal's argument and an ulp of it 3 F, which t P(t) feels by at most as much; ten steps of a polynomial whose
    # terms nearly cancel nowhere (evaluated in fp32 with both instructions an ulp off: 9 F in all, exponential included).  16 bits: the fit 20 F, the rest alike,
    # the exponent z^2 / 2 rounded twice: z^2 F.  Above 0 the same of 1 - Phi, and a rounding.
    phi = (12 * F if dtype == torch.float32 else (30 + z * z) * F) * torch.minimum(cdf, 1 - cdf) + F * (z > 0)
    e = phi * z.abs()
    want = z * cdf
    within(y, want, e + (u(dtype) + F) * (want.abs() + e) + least(dtype), "gelu")
    # the slope Phi + z phi: e^(-z^2 / 2) as above (an ulp, its correction; or z^2 F), times a constant and z
    es = phi + (8 * F if dtype == torch.float32 else (8 + z * z) * F) * z.abs() * pdf
    want = cdf + z * pdf
    within(d, want, es + (u(dtype) + F) * (want.abs() + es) + least(dtype), "slope")


@pytest.mark.parametrize("dtype", TYPES)
def test_silu_to_the_end_of_its_tail(dtype):
    z = arguments(dtype, -80, 80)
    y, d = results(z, "silu")
    z = z[:, 0].double()
    # 1 / (1 + e^-z): the exponent's constant and its product are rounded, 2 F |z|; an ulp each of exponential and reciprocal, a sum
    s = torch.sigmoid(z)
    es = (6 + 2 * z.abs()) * F * s * torch.where(z > 0, 1 - s, 1.0) + (z > 0) * 3 * F
    within(y, z * s, es * z.abs() + (u(dtype) + F) * (z * s).abs() + least(dtype), "silu")
    want = act_slope(z, "silu")
    e = (es + 4 * F * s) * (1 + z.abs())
    within(d, want, e + (u(dtype) + F) * (want.abs() + e) + least(dtype), "slope")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["leaky", "silu", "gelu"])
def test_what_is_no_number(name, dtype):
    z = torch.tensor([float("inf"), float("nan"), 1.0, -float("nan")], device="cuda", dtype=dtype)[:, None]
    y, d = results(z, name)
    assert y[0] == float("inf") and torch.isnan(y[[1, 3]]).all()
    assert torch.isfinite(y[2]) and torch.isfinite(d[2])
    if name != "leaky":
        assert torch.isnan(d[[1, 3]]).all()
    big = torch.tensor([torch.finfo(dtype).max, torch.finfo(dtype).min], device="cuda", dtype=dtype)[:, None]
    y, d = results(big, name)
    want = act(big[:, 0].double(), name)
    within(y, want, (u(dtype) + 4 * F) * want.abs(), name)
    within(d, act_slope(big[:, 0].double(), name), torch.full_like(want, 2.0 ** -20) + u(dtype), name)
