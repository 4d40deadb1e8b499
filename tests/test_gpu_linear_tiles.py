"""Every tile of aipt_linear, whole and split, with operands contiguous along either axis, and every way its results are stored."""
import pytest
import torch

from tests import linear_cases as cases
from tests.layer_util import context, empty_like_layout, generator, matrix, untouched, within
from tests.test_gpu_linear import ACTS, SLOPE, check_backward, check_forward, forward_reference

pytestmark = pytest.mark.gpu

TYPE = {4: [torch.float32], 2: [torch.bfloat16, torch.float16]}


@pytest.mark.parametrize("layout", cases.LAYOUTS, ids="-".join)
@pytest.mark.parametrize("case,dtype", [(c, t) for c in cases.FORWARD for t in TYPE[c[0]]], ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
def test_forward(case, dtype, layout):
    m, n, k = cases.sizes(case, layout)
    gen = generator(m + n + k)
    x, w, b = matrix(gen, m, k, dtype, layout[0]), matrix(gen, n, k, dtype, layout[1], scale=k ** -0.5), matrix(gen, 1, n, dtype)[0]
    way, name = cases.LAYOUTS.index(layout), ACTS[(case[1] + cases.LAYOUTS.index(layout)) % 4]
    r = matrix(gen, m, n, dtype, pad=way, offset=way)
    if way == 3:                                         # a residual in place, in rows that begin anywhere: one by one
        y, memory = empty_like_layout(m, n, dtype, "rows", 1, 1)
        y.copy_(r)
        context().linear(x, w, y, bias=b, residual=y, act=name, slope=SLOPE)
        want, bound, _, _ = forward_reference(x, w, b, r, name)
        within(y, want, bound, "y")
        assert untouched(memory, y)
    else:                                                # rows on 16 bytes where n leaves them so; from anywhere; from anywhere without the rest
        check_forward(x, w, b if way < 2 else None, r if way < 2 else None, name, pad=(0, 1, 3)[way] if n % 8 else 0, offset=(0, 1, 3)[way], keep=way < 2)


@pytest.mark.parametrize("case,dtype", [(c, t) for c in cases.BACKWARD for t in TYPE[c[0]]], ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
def test_backward(case, dtype):
    _, m, n, k = case
    gen = generator(m + n + k)
    check_backward(matrix(gen, m, n, dtype), matrix(gen, m, k, dtype), matrix(gen, n, k, dtype, scale=n ** -0.5), matrix(gen, m, n, dtype), "silu")


@pytest.mark.parametrize("dtype", TYPE[4] + TYPE[2])
def test_planar_results(dtype):
    """Pixels of planar maps: the product's transpose, whose columns are a tile's rows."""
    for m, n, k, xl in [(20000, 32, 64, "planar"), (50000, 43, 202, "planar"), (7656, 264, 488, "rows"), (3000, 520, 1032, "planar")]:
        gen = generator(m)
        x, w, b = matrix(gen, m, k, dtype, xl), matrix(gen, n, k, dtype, scale=k ** -0.5), matrix(gen, 1, n, dtype)[0]
        check_forward(x, w, b, matrix(gen, m, n, dtype, "planar"), "leaky", y_layout="planar")


@pytest.mark.parametrize("es,m,n,k,xpad,wpad", cases.ANY)
def test_lines_far_apart(es, m, n, k, xpad, wpad):
    for xl, wl in cases.any_layouts(m, k, xpad):
        for dtype in TYPE[es]:
            gen = generator(m + n)
            x, w = matrix(gen, m, k, dtype, xl, pad=xpad), matrix(gen, n, k, dtype, wl, scale=k ** -0.5, pad=wpad)
            check_forward(x, w, matrix(gen, 1, n, dtype)[0], matrix(gen, m, n, dtype), "leaky", pad=1)
            del x, w
