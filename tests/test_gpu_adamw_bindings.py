"""AdamW plans whose tensors change: graphs, bindings and streams."""
import pytest
import torch

from ai_path_tracer_denoiser_amd import api
from tests.layer_util import context, generator
from tests.test_gpu_adamw import LR, tensors

pytestmark = pytest.mark.gpu

SIZES = [5000, 3, 257]


def same(plan, other, p, q):
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    assert all(torch.equal(a.view(torch.uint8), other.state()[k].view(torch.uint8)) for k, a in plan.state().items())


@pytest.mark.parametrize("clip", [None, 0.05])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
def test_a_captured_step_keeps_the_gradients_it_was_captured_with(gtype, clip):
    gen, side = generator(40), torch.cuda.Stream()
    ctx = api.Context(0, stream=side.cuda_stream)
    p, g, new = tensors(gen, SIZES, 0.1), tensors(gen, SIZES, 0.01), tensors(gen, SIZES, 0.01, gtype)
    q = [t.clone() for t in p]
    want = context().adamw(q, [t.clone() for t in g])
    plan, graph = ctx.adamw(p, g), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        plan.update(LR, max_norm=clip)
    graph.replay()
    torch.cuda.synchronize()
    want.update(LR, max_norm=clip)
    same(plan, want, p, q)
    plan.bind(new)
    for t in g:                                          # (the graph's gradients are kept by the plan, under whatever name)
        assert any(t.data_ptr() == k.data_ptr() for k in plan._kept[0])
    del g, t
    filler = [torch.full((n,), 1e30, device="cuda") for n in SIZES for _ in range(8)]
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want.update(LR, max_norm=clip)
        same(plan, want, p, q)
    assert len(filler) == 24
    plan.update(LR, max_norm=clip)                       # and the plan itself goes on with what is bound now
    last = context().adamw(q, [t.clone() for t in new], state=want.state())
    last.update(LR, max_norm=clip)
    torch.cuda.synchronize()
    same(plan, last, p, q)


def test_a_plan_freed_while_its_steps_run():
    """Steps are queued from another current stream than the plan was made on; its memory is not given to others before they are done."""
    gen = generator(41)
    start, g = tensors(gen, SIZES, 0.1), tensors(gen, SIZES, 0.01)
    q = [t.clone() for t in start]
    want = context().adamw(q, g)
    for _ in range(3):
        want.update(LR, max_norm=1.0)
    ctx, side = api.Context(0), torch.cuda.Stream()
    p = [t.clone() for t in start]
    torch.cuda.synchronize()
    plan = ctx.adamw(p, g)
    with torch.cuda.stream(side):
        big = torch.zeros(1 << 27, device="cuda")
        for _ in range(20):
            big.add_(1.0)
        for _ in range(3):
            plan.update(LR, max_norm=1.0)
    del plan
    junk = [torch.full((k * 512,), 0xff, device="cuda", dtype=torch.uint8) for k in range(1, 60)]
    torch.cuda.synchronize()
    assert len(junk) == 59
    for a, b in zip(p, q):
        assert torch.equal(a, b)


def test_a_plan_that_outlives_its_context_or_goes_in_a_capture():
    gen = generator(42)
    p, g = tensors(gen, SIZES, 0.1), tensors(gen, SIZES, 0.01)
    ctx = api.Context(0)
    plan = ctx.adamw(p, g)
    plan.update(LR)
    ctx.close()                                          # its stream is gone
    with pytest.raises(api.AiptError, match="closed"):
        plan.update(LR)
    state = plan.state()
    del plan
    assert int(state["step"]) == 1
    del state
    side, x = torch.cuda.Stream(), torch.ones(1000, device="cuda")
    captured = api.Context(0, stream=side.cuda_stream)
    one, two = captured.adamw([t.clone() for t in p], g), captured.adamw([t.clone() for t in p], g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one.update(LR)
        two.close()
        x.add_(1)
    for k in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert int(one.state()["step"]) == k + 1 and float(x[0]) == k + 2


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_of_a_full_grid(bits, clip):
    """More than 8192 blocks of 256: every workgroup there is, several rounds each, counts itself done, replay by replay, with a step that is skipped among them."""
    gen, side = generator(43), torch.cuda.Stream()
    sizes = [3_000_001, 33, 700]
    ctx = api.Context(0, stream=side.cuda_stream)
    p, g = tensors(gen, sizes, 0.1), tensors(gen, sizes, 0.01)
    q, h = [t.clone() for t in p], [t.clone() for t in g]
    plan, eager = ctx.adamw(p, g, state_bits=bits), context().adamw(q, h, state_bits=bits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.update(LR, max_norm=clip, seed=5)
    steps = 0
    for k in range(5):
        for a, b in zip(g, h):
            a.copy_(torch.randn(a.shape, generator=gen, device="cuda") * 0.01)
            if k == 2 and clip:
                a[-1] = float("nan")
            b.copy_(a)
        graph.replay()
        eager.update(LR, max_norm=clip, seed=5)
        torch.cuda.synchronize()
        steps += not (k == 2 and clip)
        assert int(plan.state()["step"]) == int(eager.state()["step"]) == steps
        same(plan, eager, p, q)
