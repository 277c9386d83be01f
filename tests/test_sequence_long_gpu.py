"""GPU: gated leaks on rows that are split into segments of several chunks, and how exact they are over many steps."""
import pytest
import torch

from slayerpytorch_b200.recurrence import gatedLeak
from test_leak_gpu import STEP

pytestmark = pytest.mark.gpu


def warps():
    """what rows are split for: 16 an SM"""
    return torch.cuda.get_device_properties(0).multi_processor_count * 16


def segments(rows, T):
    """(segments of a row, chunks of a segment, chunks of the last one): rows of more than 512 steps, a chunk for each 512"""
    chunks = -(-(T + 3 * (T % 4 != 0)) // 512)
    if chunks < 2 or rows * 2 > warps():
        return 1, chunks, chunks
    each = -(-chunks // min(warps() // rows, chunks, 1024))
    n = -(-chunks // each)
    return n, each, chunks - (n - 1) * each


def test_no_loss_from_chunk_to_chunk():
    """Nothing is forgotten: y_t = (t + 1) x, its gradient (T - t) g.  Each sum is made in float32 over a lane's 16 steps, and five times by
    pairs of lanes; again for a chunk; five times by pairs of segments, and rounded between: less than 60 roundings of positive sums, whatever T is.
    (x is such that a sum of float32 over a segment's chunks is 120 steps off.)"""
    T = 1 << 28
    n, each, _ = segments(1, T)
    assert n > 1 and each >= 512
    v = 0.9839631
    x = torch.full((1, T), v, device="cuda", requires_grad=True)
    gate = torch.ones(1, 1, device="cuda", requires_grad=True)
    y, last = gatedLeak(x, gate, kind='decay', returnState=True)
    v = float(x.detach()[0, 0])
    t = torch.arange(T, dtype=torch.float64, device="cuda")
    off = (y.detach()[0].double() / ((t + 1) * v) - 1).abs().max()
    assert float(off) <= 60 * STEP, float(off) / STEP
    assert abs(float(last.detach()) / (T * v) - 1) <= 60 * STEP
    dx, dgate = torch.autograd.grad(y, [x, gate], torch.full_like(x, v))
    del y
    off = (dx[0].double() / ((T - t) * v) - 1).abs().max()
    assert float(off) <= 60 * STEP, float(off) / STEP
    # a product of the two for each step, added up in double
    assert abs(float(dgate) / (v * v * T * (T * T - 1) / 6) - 1) <= 130 * STEP
