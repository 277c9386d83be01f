"""GPU: gated leaks on rows that are split into segments of several chunks, and how exact they are over many steps."""
import pytest
import torch

from slayerpytorch_b200 import capi
from slayerpytorch_b200.recurrence import gatedLeak
from test_leak_gpu import STEP, TYPES, check, made

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,T,ragged", [(2, 3001, False), (2, 2048, False), (7, 8000, True), (7, 8003, True), (73, 65537, True), (600, 1000500, True)])
def test_segments_of_several_chunks(groups, T, ragged, dtype):
    """Rows of which `groups` warps fit; ragged: the last segment has fewer chunks than the others."""
    C = warps() // groups // 2
    N = 2 if C else 1
    C = max(C, 1)
    n, each, last = segments(N * C, T)
    assert n > 1 and each > 1 and (last < each) == ragged, (n, each, last)
    for shape, kind, coupled in (((N, C, T), 'logit', True), ((C, 1), 'logit', False), ((C, 1), 'decay', True)):
        x, gate, h, g, gs, gen = made(N, C, T, dtype, kind, T + N, shape)
        check(x, gate, h, None, kind, coupled, g, gs)
        lengths = torch.randint(0, T + 1, (N,), device="cuda", generator=gen)
        lengths[0] = T - 700        # ends in an earlier chunk than the row
        check(x, gate, h, lengths, kind, coupled, g, gs)


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


def pointer(v):
    return None if v is None else v.data_ptr()


def passes(x, gate, g, initial, state, gstate, dinitial, lengths=None):
    """Both passes through the C entries, rows with a gate per step: (y, state, dx, dgate, dinitial)"""
    lib, (R, T) = capi.load(), x.shape
    stream = torch.cuda.current_stream().cuda_stream
    y, dx, dgate = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    starts = torch.empty(R, lib.slayer_b200_leak_states(T), device="cuda")
    size = lib.slayer_b200_leak_workspace(R, T, 0, 0, 0)
    assert size >= 0
    room = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    args = (0, 1, R, T, pointer(lengths), 1, 0, 0, room.data_ptr(), stream)
    rc = lib.slayer_b200_leak_forward(pointer(y), pointer(state), pointer(starts), pointer(x), pointer(gate), pointer(initial), *args)
    assert rc == 0, lib.slayer_b200_last_error()
    kept = state.clone()
    rc = lib.slayer_b200_leak_backward(pointer(dx), pointer(dgate), pointer(dinitial), pointer(g), pointer(gstate), pointer(starts), pointer(x), pointer(gate), *args)
    assert rc == 0, lib.slayer_b200_last_error()
    return y, kept, dx, dgate, dinitial.clone()


@pytest.mark.parametrize("R,T", [(3, 20000), (1, 1000001), (40, 5003), (7, 700), (5000, 600), (300, 100), (1000, 5), (64, 40)])
def test_states_in_place(R, T):
    """A state that is the initial one's memory, and the gradient of the latter in the former's, whether rows are split or not."""
    gen = torch.Generator(device="cuda").manual_seed(R)
    x, gate, g = (torch.randn(R, T, device="cuda", generator=gen) for _ in range(3))
    h, up = (100 * torch.randn(R, device="cuda", generator=gen) for _ in range(2))
    gate += 6.0         # what is there at the start matters for hundreds of steps
    for lengths in (None, torch.randint(0, T + 1, (R,), device="cuda", generator=gen)):
        apart = passes(x, gate, g, h, torch.empty_like(h), up, torch.empty_like(h), lengths)
        y, state = gatedLeak(x, gate, initial=h, lengths=lengths, returnState=True)
        assert torch.equal(apart[0], y) and torch.equal(apart[1], state)
        for _ in range(5):
            own, back = h.clone(), up.clone()
            assert all(torch.equal(a, b) for a, b in zip(apart, passes(x, gate, g, own, own, back, back, lengths)))


@pytest.mark.parametrize("T", [300, 480, 2000])
def test_a_decay_of_a_whole_row_is_not_rounded_again_at_each_step(T):
    """Rows whose f lies 0.4 to 0.5 of a rounding step, 2^-24, below a float32 number: where steps took f so rounded, a lane's 16 of them would forget
    too little each time, and results were 3 to 4 STEP too large on average.  Decays themselves are off by 6 STEP of 1 - f at most, of any sign: on
    average over 64 of them hardly by one.  What steps round goes either way."""
    grid = torch.linspace(3.0, 6.0, 100000)
    small = torch.sigmoid(-grid.double()).float().double()
    up = ((1.0 - small).float().double() - (1.0 - small)) / STEP
    gate = grid[(up > 0.4) & (up < 0.5)]
    gate = gate[torch.linspace(0, len(gate) - 1, 64).long()]
    gen = torch.Generator(device="cuda").manual_seed(T)
    x, g = (0.5 + torch.rand(8, 64, T, device="cuda", generator=gen) for _ in range(2))
    leaves = [x.requires_grad_(), gate[:, None].cuda().requires_grad_()]
    y = gatedLeak(*leaves)
    dx, dgate = torch.autograd.grad(y, leaves, g)
    f = torch.sigmoid(leaves[1].detach().double())[None]

    def scan(v):
        out, h = torch.empty_like(v), torch.zeros_like(v[..., 0])
        for t in range(T):
            h = f[..., 0] * h + v[..., t]
            out[..., t] = h
        return out
    h, lam = scan(x.detach().double()), scan(g.double().flip(-1)).flip(-1)
    slope = (lam * f * (1 - f) * torch.cat([torch.zeros_like(h[..., :1]), h[..., :-1]], -1)).sum((0, 2))[:, None]
    off = [float((a.double() / b - 1).mean()) / STEP for a, b in ((y.detach(), h), (dx, lam), (dgate, slope))]
    assert abs(off[0]) <= 2 and abs(off[1]) <= 2 and abs(off[2]) <= 4, off
