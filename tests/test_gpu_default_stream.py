"""Traces, frames, batches and prefetches of a context on HIP's default stream: the bits of a context on a stream of its own."""
import numpy as np
import pytest
import torch

from ai_path_tracer_denoiser_amd import api, synth
from tests.test_gpu_frame import _mesh_scene

pytestmark = pytest.mark.gpu

W, H, DEPTH, FRAMES = 320, 192, 4, 7


def run(stream, batch, prefetch):
    """Outputs, G-buffers and live counts of seven frames, and a trace of two frames by itself."""
    sc, mats, faces, box = _mesh_scene((W, H), DEPTH)
    cams = [sc.orbit(phi=sc.phi + 0.1 * k) for k in range(FRAMES)]
    side = torch.cuda.Stream() if stream == "torch" else None
    ctx = api.Context(0, stream=side.cuda_stream if side else stream)
    ctx.pathtrace_init(sc.geoms, mats, faces, box)
    ctx.load_weights(synth.make_blob(7))
    ctx.frame_configure(W, H)
    if batch > 1:
        ctx.frames_configure(batch)
    out, gbufs, k = [torch.empty(3, H, W, device="cuda") for _ in range(batch)], [], 0
    torch.cuda.synchronize()
    frames = []
    while k < FRAMES:
        nb = min(batch, FRAMES - k)
        if batch == 1:
            ctx.frame(cams[k], 1, DEPTH, out[0], bn_batch=True, carry=k > 0)
            if prefetch and k + 1 < FRAMES:
                ctx.frame_prefetch(cams[k + 1], 1, DEPTH)
        else:
            ctx.frames(cams[k:k + nb], 1, DEPTH, out, bn_batch=True, carry_first=k > 0, carry=True)
            if prefetch and k + nb < FRAMES:
                ctx.frames_prefetch(cams[k + nb:k + nb + min(batch, FRAMES - k - nb)], 1, DEPTH)
        ctx.sync()
        ptr, rows, stride = ctx.gbuffer()
        host = np.empty((10, rows, stride), np.float32)
        assert api.lib().aipt_download(ctx._h, host.ctypes.data, ptr, host.nbytes) == 0
        gbufs.append(host)
        frames += [o.cpu().numpy().copy() for o in out[:nb]]
        k += nb
    ctx.close()
    return frames, gbufs


@pytest.mark.parametrize("batch,prefetch", [(1, False), (1, True), (4, False), (3, True)])
def test_every_stream_gives_the_same_frames(batch, prefetch):
    want, gbufs = run(None, batch, prefetch)
    assert len(want) == FRAMES and all(np.isfinite(f).all() for f in want)
    for stream in (api.STREAM_DEFAULT, "torch"):
        frames, g = run(stream, batch, prefetch)
        for k in range(FRAMES):
            assert np.array_equal(frames[k], want[k]), (stream, k)
        for k, (a, b) in enumerate(zip(g, gbufs)):
            assert np.array_equal(a, b), (stream, "gbuffer", k)


def test_torch_reads_frames_of_the_default_stream_without_waiting():
    """On the default stream torch's own work follows the frame's, in order, and the next frame follows that."""
    sc, mats, faces, box = _mesh_scene((W, H), DEPTH)
    cams = [sc.orbit(phi=sc.phi + 0.1 * k) for k in range(FRAMES)]
    want, _ = run(None, 1, False)
    ctx = api.Context(0, stream=api.STREAM_DEFAULT)
    ctx.pathtrace_init(sc.geoms, mats, faces, box)
    ctx.load_weights(synth.make_blob(7))
    ctx.frame_configure(W, H)
    out, kept = torch.empty(3, H, W, device="cuda"), []
    for k in range(FRAMES):
        ctx.frame(cams[k], 1, DEPTH, out, bn_batch=True, carry=k > 0)
        kept.append(out.clone())
    ctx.sync()
    for k in range(FRAMES):
        assert np.array_equal(kept[k].cpu().numpy(), want[k]), k
