"""Sizes that send aipt_linear to each of its kernels, and what is to be launched for them: a change of the estimate that chooses must not leave one untested.

FORWARD: (element size, tile rows, tile columns, bytes a lane loads, is the contraction split) -> (m, n, k).  With k several times round the ring of LDS slots, and
a remainder; m and n no multiples of a tile; operands contiguous along either axis.  Where loads are of 16 bytes, an axis that is not
contiguous in memory is made odd (`sizes`)."""
import ctypes as C

from ai_path_tracer_denoiser_amd import api

FORWARD = {
    (4, 64, 64, 4, False): (2526, 73, 255), (4, 64, 64, 4, True): (557, 66, 6774), (4, 64, 64, 16, False): (440, 80, 232), (4, 64, 64, 16, True): (880, 400, 496),
    (4, 128, 128, 16, False): (344, 8224, 248), (4, 128, 128, 16, True): (216, 4120, 1688), (4, 256, 32, 4, False): (17226, 65, 251), (4, 256, 32, 4, True): (1885, 66, 2386),
    (4, 256, 32, 16, False): (17336, 80, 232), (4, 256, 32, 16, True): (8456, 72, 496), (4, 256, 64, 16, False): (39704, 136, 248), (4, 256, 64, 16, True): (3280, 304, 2008),
    (4, 256, 256, 16, True): (456, 6232, 2840),
    (2, 64, 64, 4, False): (100, 118, 468), (2, 64, 64, 4, True): (1034, 198, 1394), (2, 64, 64, 16, False): (104, 104, 464), (2, 64, 64, 16, True): (1632, 72, 1872),
    (2, 128, 128, 16, False): (9976, 264, 472), (2, 128, 128, 16, True): (5528, 136, 4960), (2, 256, 32, 4, False): (35156, 86, 506), (2, 256, 32, 4, True): (8694, 70, 3002),
    (2, 256, 32, 16, False): (50496, 40, 472), (2, 256, 32, 16, True): (8240, 72, 4128), (2, 256, 64, 16, False): (37192, 136, 472), (2, 256, 64, 16, True): (5576, 144, 6664),
    (2, 256, 256, 16, False): (7656, 1544, 480), (2, 256, 256, 16, True): (592, 6608, 4208),
}
LAYOUTS = [("rows", "rows"), ("rows", "planar"), ("planar", "rows"), ("planar", "planar")]      # of x and w
# (element size, m, n, k) -> tiles and splits of dx and of dw
BACKWARD = {
    (2, 505, 712, 4136): ((64, 64, False), (128, 128, False)), (2, 8149, 4120, 72): ((64, 64, False), (128, 128, True)), (2, 9857, 4344, 136): ((64, 64, False), (256, 32, True)),
    (2, 10081, 4224, 152): ((64, 64, False), (256, 64, True)), (2, 511, 4440, 2792): ((64, 64, False), (256, 256, False)), (2, 16963, 4632, 144): ((256, 256, True), (256, 256, True)),
    (2, 27661, 384, 72): ((128, 128, False), (64, 64, True)), (2, 6263, 4512, 72): ((128, 128, True), (64, 64, True)), (2, 18081, 400, 136): ((256, 32, False), (64, 64, True)),
    (2, 34753, 400, 136): ((256, 64, False), (64, 64, True)), (2, 25915, 392, 392): ((256, 256, False), (64, 64, True)), (2, 203, 72, 136): ((64, 64, False), (64, 64, False)),
    (4, 511, 776, 4328): ((64, 64, False), (128, 128, False)), (4, 3635, 72, 4952): ((64, 64, False), (128, 128, True)), (4, 515, 3600, 536): ((64, 64, True), (256, 32, False)),
    (4, 1757, 208, 4632): ((256, 64, False), (256, 64, True)), (4, 1351, 192, 2816): ((128, 128, False), (64, 64, True)), (4, 8767, 1568, 104): ((128, 128, True), (64, 64, True)),
    (4, 12851, 2992, 208): ((256, 256, True), (256, 32, True)), (4, 203, 72, 136): ((64, 64, False), (64, 64, False)),
}


# (element size, m, n, k, pads of x's and w's lines) -> lines so far apart, or so long and unaligned, that each load is checked for itself
ANY = [(4, 70, 30, 5, 1 << 21, 0), (4, 70, 30, 25, 1 << 21, 1 << 21), (4, 200, 3, 600, 1 << 21, 3), (2, 2, 3, (1 << 22) + 9, 0, 0), (2, 3, 2, (1 << 22) + 9, 0, 4), (2, (1 << 22) + 9, 3, 5, 0, 0)]


def any_layouts(m, k, xpad):
    """Long lines are long along the contraction, or along the pixels of planar maps."""
    return LAYOUTS if xpad else [("rows", "rows")] if k > m else [("planar", "rows"), ("planar", "planar")]


def sizes(case, layout):
    """The case's sizes, an axis odd where that leaves lines on 16 bytes."""
    m, n, k = FORWARD[case]
    return (m, n, k) if case[3] == 4 else (m + 3 * (layout[0] == "rows"), n + 5 * (layout[1] == "rows"), k)


def strides(at, rows, cols, layout="rows", pad=0):
    return (at, cols + pad, 1) if layout == "rows" else (at, 1, rows + pad)


def forward_plan(type, m, n, k, xl, wl, yl="rows", xpad=0, wpad=0):
    plan, p = api.LinearPlan(), 1 << 40
    record = api._LINEAR.pack(type, 0, 0.1, 0, m, n, k, *strides(p, m, k, xl, xpad), *strides(2 * p, n, k, wl, wpad), *strides(3 * p, m, n, yl), 0, 0, 0, 0, 0, 0, 0)
    assert api.lib().aipt_linear_planned(None, record, C.byref(plan)) == 0
    return plan


def backward_plan(type, act, m, n, k):
    dx, dw, p = api.LinearPlan(), api.LinearPlan(), 1 << 40
    z = (4 * p, n, 1) if act else (0, 0, 0)
    record = api._LINEAR_GRAD.pack(type, act, 0.1, 0, m, n, k, p, n, 1, 2 * p, k, 1, 3 * p, k, 1, *z, 5 * p, k, 1, 6 * p, k, 1, 7 * p)
    assert api.lib().aipt_linear_backward_planned(None, record, C.byref(dx), C.byref(dw)) == 0
    return dx, dw
