"""Gradients of the layer operators where something is infinite or no number: what it enters, and nothing else."""
import pytest
import torch

from tests.layer_util import TYPES, context, generator, matrix, u

pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)


def same_but(clean, odd, hit):
    """Equal to the last bit where `hit` is not, not finite where it is."""
    assert torch.equal(bits(clean)[~hit], bits(odd)[~hit]) and not torch.isfinite(odd[hit]).any() and torch.isfinite(clean).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(dtype, bad):
    for m, n, k, name in [(130, 70, 200, "none"), (131, 71, 201, "silu"), (9000, 40, 24, "gelu"), (3, 1000, 520, "leaky")]:
        for where in ("dy", "preact"):
            if where == "preact" and (name == "none" or (name == "leaky" and bad == bad) or bad > 0):      # a slope of +inf is 1 or no number, as the formula has it
                continue
            outs = []
            for spoil in (False, True):
                gen = generator(m + n)
                dy, x, w, z = matrix(gen, m, n, dtype), matrix(gen, m, k, dtype), matrix(gen, n, k, dtype, scale=n ** -0.5), matrix(gen, m, n, dtype)
                i, j = m - 1, n - 2
                dy[i, j] = 1.0
                if spoil:
                    (dy if where == "dy" else z)[i, j] = bad
                dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda", dtype=dtype)
                context().linear_backward(dy, x, w, preact=None if name == "none" else z, act=name, dx=dx, dw=dw, dbias=db)
                outs.append((dx, dw, db))
            row, line, one = torch.zeros(m, dtype=torch.bool, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
            if where == "preact" and name == "leaky":
                continue                                 # (a NaN pre-activation is not above 0: the slope's)
            row[i], line[j], one[j] = True, True, True
            for clean, odd, hit in zip(*outs, (row, line, one)):
                same_but(clean, odd, hit)


def test_half_precision_overflows_to_infinity_and_nothing_else():
    """dz is rounded to the type: 60000 times GELU's steepest slope, 1.129, is none of fp16's numbers, 57000 times it is.  bf16 and fp32 hold both."""
    z = torch.full((64, 8), 1.414, device="cuda")
    x, w = torch.full((64, 16), 1e-3, device="cuda"), torch.full((8, 16), 1e-3, device="cuda")
    for dtype in TYPES:
        for size in (57000.0, 60000.0):
            dy, dx, dw = torch.full((64, 8), size, device="cuda").to(dtype), torch.empty(64, 16, device="cuda", dtype=dtype), torch.empty(8, 16, device="cuda", dtype=dtype)
            context().linear_backward(dy, x.to(dtype), w.to(dtype), preact=z.to(dtype), act="gelu", dx=dx, dw=dw)
            if dtype == torch.float16 and size == 60000.0:
                assert torch.isinf(dx).all() and torch.isinf(dw).all()
            else:
                # slope within 1.1289 (1 +- 2^-9), three roundings of operands, one of dz, one of the result
                for got, terms in ((dx, 8), (dw, 64)):
                    assert bool(((got.double() / (1.1289 * size * 1e-3 * terms) - 1).abs() < 6 * u(dtype) + 2e-3).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", TYPES)
def test_block_norm(dtype, kind, bad):
    for m, c, groups in [(24, 80, 3), (1500, 57, 5), (40, 2048, 2), (1200, 33, 600)]:
        for where in ("dh", "dz"):
            outs = []
            for spoil in (False, True):
                gen = generator(c)
                y, x, dh, dz = (matrix(gen, m, c, dtype) for _ in range(4))
                gate = matrix(gen, groups, c, dtype)
                vec = {k: matrix(gen, 1, c, dtype)[0] for k in ("scale", "post_weight", "pre_weight")}
                bias = {"post_bias": matrix(gen, 1, c, dtype)[0]} if kind == "layer" else {}
                h, z, st = torch.empty_like(x), torch.empty_like(x), torch.empty(m, 4, device="cuda")
                context().block_norm(y, x, h, z, gate=gate, kind=kind, stats=st, **vec, **bias)
                i, j = m - 2, c // 2
                if spoil:
                    (dh if where == "dh" else dz)[i, j] = bad
                dx, dy, dgate = torch.empty_like(x), torch.empty_like(x), torch.empty_like(gate)
                grads = {"d" + k: torch.empty_like(v) for k, v in vec.items()}
                if kind == "layer":
                    grads.update(dpost_bias=torch.empty(c, device="cuda", dtype=dtype), dpre_bias=torch.empty(c, device="cuda", dtype=dtype))
                context().block_norm_backward(dh, dz, y, h, st, gate=gate, kind=kind, dx=dx, dy=dy, dgate=dgate, **vec, **bias, **grads)
                outs.append({"dx": dx, "dy": dy, "dgate": dgate, **grads})
            clean, odd = outs
            row, group = torch.zeros(m, dtype=torch.bool, device="cuda"), torch.zeros(groups, dtype=torch.bool, device="cuda")
            row[i], group[i // (m // groups)] = True, True
            cell = torch.zeros(c, dtype=torch.bool, device="cuda")
            cell[j] = True
            for k in ("dx", "dy"):
                assert torch.equal(bits(clean[k])[~row], bits(odd[k])[~row])
            assert not torch.isfinite(odd["dy"][row]).any()
            assert torch.equal(bits(clean["dgate"])[~group], bits(odd["dgate"])[~group])
            if where == "dh":                            # it enters its own column of dx, and through the norm behind the block all of the row's dy
                same_but(clean["dx"][row], odd["dx"][row], cell[None])
                same_but(clean["dgate"][group], odd["dgate"][group], cell[None])
                for k in set(grads) - {"dpre_weight", "dpre_bias"}:
                    same_but(clean[k], odd[k], cell)
                for k in set(grads) & {"dpre_weight", "dpre_bias"}:
                    assert torch.equal(bits(clean[k]), bits(odd[k]))
            else:                                        # through the norm before the next block all of the row's dx
                assert not torch.isfinite(odd["dx"][row]).any() and not torch.isfinite(odd["dgate"][group]).any()
                for k in set(grads) & {"dpre_weight", "dpre_bias"}:
                    same_but(clean[k], odd[k], cell)
                for k in set(grads) - {"dpre_weight", "dpre_bias"}:
                    assert not torch.isfinite(odd[k]).any()
