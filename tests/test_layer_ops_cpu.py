"""What the layer operators refuse, on the C boundary and in the binding: no GPU is needed to be told."""
import ctypes as C

import pytest
import torch

from ai_path_tracer_denoiser_amd import api

P = 1 << 20          # an address nobody follows


def error(rc):
    assert rc == -1
    return api.lib().aipt_last_error(None).decode()


def linear(type=0, act=0, slope=0.1, reserved=0, m=8, n=6, k=4, x=(P, 4, 1), w=(2 * P, 4, 1), y=(3 * P, 6, 1), residual=(0, 0, 0), preact=(0, 0, 0), bias=0):
    return api._LINEAR.pack(type, act, slope, reserved, m, n, k, *x, *w, *y, *residual, *preact, bias)


def linear_grad(type=0, act=0, slope=0.1, reserved=0, m=8, n=6, k=4, dy=(P, 6, 1), x=(2 * P, 4, 1), w=(3 * P, 4, 1), preact=(0, 0, 0), dx=(4 * P, 4, 1), dw=(5 * P, 4, 1), dbias=6 * P):
    return api._LINEAR_GRAD.pack(type, act, slope, reserved, m, n, k, *dy, *x, *w, *preact, *dx, *dw, dbias)


@pytest.mark.parametrize("bad,word", [
    (dict(type=3), "type"), (dict(act=4), "act"), (dict(act=-1), "act"), (dict(slope=float("nan")), "slope"), (dict(reserved=1), "reserved"), (dict(m=-1), "sizes"),
    (dict(n=1 << 31), "sizes"), (dict(x=(0, 4, 1)), "x is NULL"), (dict(w=(0, 4, 1)), "w is NULL"), (dict(y=(0, 6, 1)), "y is NULL"), (dict(x=(P + 2, 4, 1)), "misaligned"),
    (dict(x=(P, 8, 2)), "x: strides"), (dict(w=(P, -4, 1)), "w: strides"), (dict(y=(3 * P, 5, 1)), "y: strides"), (dict(y=(3 * P, 0, 1)), "y: strides"), (dict(y=(3 * P, 1, 7)), "y: strides"),
    (dict(y=(P, 6, 1)), "overlaps an input"), (dict(y=(2 * P + 64, 6, 1)), "overlaps an input"), (dict(preact=(3 * P, 6, 1)), "outputs overlap"), (dict(bias=3 * P + 4), "overlaps an input"),
    (dict(residual=(3 * P + 24, 6, 1)), "overlaps the residual"), (dict(residual=(3 * P, 7, 1)), "overlaps the residual"), (dict(bias=5 * P + 1), "bias is misaligned"), (dict(), "ctx is NULL"),
    (dict(residual=(3 * P, 6, 1)), "ctx is NULL"),                                             # the residual may be y itself
    (dict(x=(P, 20, 1), y=(P + 16, 20, 1), n=6, k=4), "ctx is NULL"),                          # windows side by side in the rows of one buffer
    (dict(x=(P, 20, 1), y=(P + 12, 20, 1), n=6, k=4), "overlaps an input"), (dict(x=(P, 0, 1)), "ctx is NULL"), (dict(y=(3 * P, 1, 8)), "ctx is NULL"),
    (dict(m=0, x=(0, 4, 1), y=(0, 6, 1)), "ctx is NULL"),
])
def test_linear_refuses(bad, word):
    assert word in error(api.lib().aipt_linear(None, linear(**bad), None, 0))


def test_workspace_is_asked_for_and_checked():
    need = C.c_size_t()
    big = dict(m=64, n=64, k=100000, x=(P, 100000, 1), w=(1 << 30, 100000, 1), y=(1 << 32, 64, 1))
    assert api.lib().aipt_linear_workspace(None, linear(**big), C.byref(need)) == 0 and need.value > 0
    assert "workspace" in error(api.lib().aipt_linear(None, linear(**big), None, 0))
    assert "workspace" in error(api.lib().aipt_linear(None, linear(**big), 1 << 34, need.value - 1))
    assert "workspace" in error(api.lib().aipt_linear(None, linear(**big), (1 << 34) + 4, need.value))
    assert "ctx is NULL" in error(api.lib().aipt_linear(None, linear(**big), 1 << 34, need.value))
    assert "overlap" in error(api.lib().aipt_linear(None, linear(**big), 1 << 32, need.value))
    assert "bytes is NULL" in error(api.lib().aipt_linear_workspace(None, linear(), None))


@pytest.mark.parametrize("bad,word", [
    (dict(type=-1), "type"), (dict(act=1), "preact is NULL"), (dict(dy=(0, 6, 1)), "dy is NULL"), (dict(x=(0, 4, 1)), "x is NULL"), (dict(w=(0, 4, 1)), "w is NULL"),
    (dict(dx=(4 * P, 3, 1)), "dx: strides"), (dict(dw=(4 * P + 32, 4, 1)), "outputs overlap"), (dict(dx=(P, 4, 1)), "overlaps an input"), (dict(dbias=P + 4), "overlaps an input"),
    (dict(dbias=6 * P + 2), "dbias is misaligned"), (dict(dy=(P, 12, 2)), "dy: strides"), (dict(dbias=0), "ctx is NULL"), (dict(dx=(0, 0, 0), w=(0, 0, 0), dbias=0), "ctx is NULL"),
])
def test_linear_backward_refuses(bad, word):
    a = linear_grad(**bad)
    need = C.c_size_t()
    api.lib().aipt_linear_backward_workspace(None, a, C.byref(need))
    assert word in error(api.lib().aipt_linear_backward(None, a, 1 << 40, need.value))


def norm(type=0, kind=0, eps=1e-5, c=8, rows=6, groups=1, x=P, y=2 * P, h=3 * P, z=4 * P, strides=(8, 8, 8, 8), gate=0, scale=0, w1=0, b1=0, w2=0, b2=0, stats=0):
    return api._NORM.pack(type, kind, eps, c, rows, groups, x, y, h, z, *strides, gate, scale, w1, b1, w2, b2, stats)


@pytest.mark.parametrize("bad,word", [
    (dict(type=9), "type"), (dict(kind=2), "kind"), (dict(c=0), "channels"), (dict(c=16385), "channels"), (dict(rows=-1), "rows"), (dict(groups=4, gate=9 * P), "groups"), (dict(groups=0), "groups"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(b1=5 * P), "AIPT_NORM_LAYER"), (dict(b2=5 * P), "AIPT_NORM_LAYER"), (dict(y=0, scale=5 * P), "belong to a block"),
    (dict(z=0, w2=5 * P), "pre_* belong"), (dict(x=0), "NULL"), (dict(h=0), "NULL"), (dict(strides=(8, 8, 7, 8)), "row strides"), (dict(strides=(-8, 8, 8, 8)), "row strides"),
    (dict(x=P + 2), "misaligned"), (dict(stats=7 * P + 4), "stats"), (dict(z=3 * P), "outputs overlap"), (dict(h=2 * P), "overlaps an input"), (dict(z=P), "overlaps an input"), (dict(scale=3 * P), "overlaps an input"),
    (dict(h=P, strides=(9, 8, 8, 8)), "overlaps an input"), (dict(h=P), "ctx is NULL"), (dict(groups=3, gate=9 * P), "ctx is NULL"), (dict(rows=0, x=0), "ctx is NULL"), (dict(kind=1, b1=5 * P), "ctx is NULL"),
])
def test_block_norm_refuses(bad, word):
    assert word in error(api.lib().aipt_block_norm(None, norm(**bad)))


def norm_grad(type=0, kind=0, c=8, reserved=0, rows=6, groups=1, dh=P, dz=2 * P, y=3 * P, h=4 * P, stats=5 * P, gate=0, scale=0, w1=0, b1=0, w2=0, dx=6 * P, dy=7 * P, strides=(8,) * 6, dgate=0,
              dscale=0, dw1=0, db1=0, dw2=0, db2=0):
    return api._NORM_GRAD.pack(type, kind, c, reserved, rows, groups, dh, dz, y, h, stats, gate, scale, w1, b1, w2, dx, dy, *strides, dgate, dscale, dw1, db1, dw2, db2)


@pytest.mark.parametrize("bad,word", [
    (dict(reserved=1), "reserved"), (dict(c=0), "channels"), (dict(dh=0, dz=0), "neither"), (dict(stats=0), "stats is NULL"), (dict(h=0), "dz without h"), (dict(y=0), "belong to a block"),
    (dict(dz=0, dw2=8 * P), "pre_* belong"), (dict(db1=8 * P), "AIPT_NORM_LAYER"), (dict(dx=2 * P), "overlaps an input"), (dict(dy=6 * P), "outputs overlap"), (dict(dscale=7 * P + 4), "outputs overlap"),
    (dict(strides=(8, 8, 8, 8, 7, 8)), "row strides"), (dict(strides=(8, -8, 8, 8, 8, 8)), "row stride"), (dict(groups=5, dgate=8 * P), "groups"), (dict(dx=P), "ctx is NULL"), (dict(dgate=8 * P, groups=2), "ctx is NULL"),
    (dict(stats=5 * P + 8), "aligned"),
])
def test_block_norm_backward_refuses(bad, word):
    a = norm_grad(**bad)
    need = C.c_size_t()
    api.lib().aipt_block_norm_backward_workspace(None, a, C.byref(need))
    assert word in error(api.lib().aipt_block_norm_backward(None, a, 1 << 40, need.value))
    if bad.get("dgate") and word == "ctx is NULL":
        assert "workspace" in error(api.lib().aipt_block_norm_backward(None, a, None, 0))


def test_adamw_counts():
    def of(fn, *counts):
        return fn((C.c_longlong * max(1, len(counts)))(*counts), len(counts))
    L = api.lib()
    assert [of(L.aipt_adamw_state_elements, *c) for c in ((), (0,), (1,), (256, 257), (3, 0, 1000))] == [0, 0, 256, 768, 256 + 1024]
    assert of(L.aipt_adamw_state_elements, -1) < 0 and of(L.aipt_adamw_state_elements, 1 << 41) < 0 and of(L.aipt_adamw_workspace, -1) < 0
    assert of(L.aipt_adamw_workspace, 10) >= 256 + 4 and of(L.aipt_adamw_workspace, *([5] * 1000)) >= 256 + 4 * 9 * 2


def adamw(param=P, grad=2 * P, copy=0, count=300, decay=0.01, grad_type=0, copy_type=1, bits=32, m=3 * P, v=4 * P, ms=None, vs=None, step=5 * P, norm=6 * P, ws=7 * P, size=1 << 19, n=1):
    h = C.c_void_p()
    return api.lib().aipt_adamw_create(None, api._ADAMW_TENSOR.pack(param, grad, copy, count, decay, 0), n, grad_type, copy_type, bits, m, v, ms, vs, step, norm, ws, size, C.byref(h))


@pytest.mark.parametrize("bad,word", [
    (dict(n=-1), "tensors"), (dict(grad_type=5), "grad_type"), (dict(copy_type=0), "copy_type"), (dict(bits=16), "state_bits"), (dict(param=0), "NULL param"), (dict(count=-1), "elements"),
    (dict(decay=float("inf")), "weight_decay"), (dict(m=None), "m or v"), (dict(bits=8), "m_scale"), (dict(step=None), "NULL"), (dict(ws=None), "NULL"), (dict(param=P + 1), "misaligned"),
    (dict(m=3 * P + 4), "aligned"), (dict(grad=P), "overlaps"), (dict(grad=P + 1196), "overlaps"), (dict(copy=2 * P + 8), "overlaps"), (dict(v=3 * P + 16), "overlaps"), (dict(step=P + 8), "overlaps"),
    (dict(ws=6 * P), "overlaps"), (dict(), "ctx is NULL"), (dict(grad=P + 1200), "ctx is NULL"),
])
def test_adamw_refuses(bad, word):
    assert word in error(adamw(**bad))
    assert "no plan" in error(api.lib().aipt_adamw_step(None, None, 1e-3, .9, .999, 1e-8, 0.0, 0))
    api.lib().aipt_adamw_destroy(None)


def test_binding_refuses():
    ctx = api.Context.__new__(api.Context)
    ctx._h, ctx.device = None, 0
    x = torch.zeros(4, 4)
    for call in (lambda: ctx.linear(x, x, x), lambda: ctx.linear_backward(x, x, x), lambda: ctx.block_norm(None, x, x), lambda: ctx.block_norm_backward(x, None, None, None, None),
                 lambda: ctx.linear(x.double(), x, x)):
        with pytest.raises(api.AiptError, match="is wanted"):
            call()
    with pytest.raises(api.AiptError, match="one of"):
        api._choice("act", "relu", api.ACTIVATIONS)
