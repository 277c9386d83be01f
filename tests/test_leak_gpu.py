"""GPU: the gated leaky integrator against the recurrence in double.

Tolerances, in steps of S = 2^-24.
f = sigmoid(gate): e = 2^z, z = -|gate| log2(e), is off by half a step of z, |gate| S at most, and 4 S of the power itself; 1 + e, its
reciprocal and their product add 4 S: the smaller of f and 1 - f is off by D = (8 + |gate|) S of itself.
A lane's map of up to 16 steps: f is rounded once more and each step rounds once, so that what is added (B) is off by 32 S of its terms'
magnitudes, the product A of f's by 32 S of itself, R = 1 - A by 48 S.  Composing two maps, R is off by r (R1 + R2) / (R1 + R2 - R1 R2) + 2, at
most 1.4 times as much while it is used (below 1/2), A by what R is or, beyond, by the sum of both, which is less than the same multiple of
what the steps forget; B by what is lost of the first map's.  So all of it is as if each step forgot, and added, 160 S of itself too much or
too little: followed along the recurrence (`want`) with magnitudes that no sign cancels.  The walk of up to 16 steps from a lane's state
rounds f and the result, 3 S of the largest state each time.  States between calls and for the backward pass are 32 bits, differences and
products there are rounded once.  A result is rounded to its type: half a step of it, and S on the way through float32."""
import pytest
import torch

from slayerpytorch_b200 import layer
from slayerpytorch_b200.recurrence import gatedLeak, gatedLeakStep

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP = 2.0 ** -24
MAPS = 160 * STEP


def scan(f, u, first):
    """h_t = f_t h_{t-1} + u_t from `first` on, in double: steps composed by doubling"""
    f, h = f.clone(), u.clone()
    if f.shape[1] == 0:
        return h
    h[:, 0] += f[:, 0] * first
    k = 1
    while k < f.shape[1]:
        h[:, k:] += f[:, k:] * h[:, :-k].clone()
        f[:, k:] = f[:, k:] * f[:, :-k].clone()
        k *= 2
    return h


def shifted(h, first):
    return torch.cat([first[:, None], h[:, :-1]], 1)


def window(v):
    """sums over a step and the 16 before it"""
    total = torch.nn.functional.pad(v, (17, 0)).cumsum(1)
    return total[:, 17:] - total[:, :-17] + 1e-12 * total[:, -1:]


def want(x, gate, initial, lengths, kind, coupled, g=None, gstate=None):
    """(value, bound) of y, the last state and, with g, the gradients of x, gate (per step) and initial; rows [R, T], in double"""
    x, gate = x.double(), gate.double().expand(x.shape)
    R, T = x.shape
    f = torch.sigmoid(gate) if kind == 'logit' else gate
    rest = torch.sigmoid(-gate) if kind == 'logit' else 1.0 - gate
    D = (8 + gate.abs()) * STEP if kind == 'logit' else torch.full_like(f, STEP)
    off, offr = (D + MAPS) * torch.minimum(f, rest), D * torch.minimum(f, rest) + STEP * rest
    on = torch.arange(T, device=x.device)[None] < (torch.full((R,), T, device=x.device) if lengths is None else lengths)[:, None]
    x = torch.where(on, x, 0.0)
    u = rest * x if coupled else x
    offu = MAPS * u.abs() + (offr * x.abs() + STEP * u.abs() if coupled else 0.0)
    zero = torch.zeros(R, dtype=torch.float64, device=x.device)
    h0 = zero if initial is None else initial.double()
    keep = torch.where(on, f, 1.0)                       # behind a length the state stays what it is
    h = scan(keep, torch.where(on, u, 0.0), h0)
    size = scan(keep, torch.where(on, u.abs(), 0.0), h0.abs())
    before = shifted(h, h0)
    e = scan(keep, torch.where(on, off * shifted(size, h0.abs()) + offu, 0.0), zero)
    walk = 3 * STEP * (window(size) + h0.abs()[:, None])
    out = [(h * on, (e + walk) * on), (h[:, -1], e[:, -1])]
    if g is None:
        return out
    g = torch.where(on, g.double(), 0.0)
    gs = zero if gstate is None else gstate.double()
    # c_t = f_t (g_t + c_{t+1}): what step t hands back
    c = scan(keep.flip(1), (keep * g).flip(1), gs).flip(1)
    csize = scan(keep.flip(1), (keep * g.abs()).flip(1), gs.abs()).flip(1)
    after = lambda v, last: torch.cat([v[:, 1:], last[:, None]], 1)  # noqa: E731
    lam, lsize = g + after(c, gs), g.abs() + after(csize, gs.abs())
    ec = scan(keep.flip(1), torch.where(on, off * lsize + MAPS * f * g.abs(), 0.0).flip(1), zero).flip(1)
    el = after(ec, zero) + 3 * STEP * (window(lsize.flip(1)).flip(1) + gs.abs()[:, None])
    # a state of 32 bits at a chunk's start, carried on
    eb = shifted(e + walk, zero) + 2 * STEP * torch.maximum(before.abs().amax(1, keepdim=True), size)
    r = rest if coupled else torch.ones_like(rest)
    dx, edx = lam * r, el * r.abs() + lam.abs() * ((offr if coupled else 0.0) + STEP * r.abs())
    d = before - x if coupled else before
    ed = eb + STEP * d.abs()
    m = f * rest if kind == 'logit' else torch.ones_like(f)
    dg, edg = lam * d * m, (el * d.abs() + lam.abs() * ed) * m.abs() + (2 * D + 6 * STEP) * (lam * d * m).abs()
    return out + [(dx * on, edx * on), (dg * on, edg * on), (c[:, 0], ec[:, 0])]


def close(got, value, bound):
    half = torch.finfo(got.dtype).eps / 2
    limit = bound * (1 + half) + (half + STEP) * value.abs() + 2.0 ** -24 * (got.dtype == torch.float16) + 1e-37
    # what lies beyond the type's largest number (float16: 65504, and half a step of 16) is an infinity in it
    beyond = value.abs() - limit > torch.finfo(got.dtype).max
    value, got = torch.where(beyond, value.sign(), value), torch.where(beyond & got.isinf(), got.sign().double(), got.double())
    wrong = (got - value).abs() - limit
    assert got.shape == value.shape and bool((wrong <= 0).all()), "off by %g beyond the limit, of %g" % (wrong.max(), value.abs().max())


def made(N, C, T, dtype, kind, seed, shape=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    x = rand(N, C, T).to(dtype)
    gate = rand(*(shape or (N, C, T))) * 2 + 1.5
    gate = (torch.sigmoid(gate) if kind == 'decay' else gate).to(dtype)
    return x, gate, rand(N, C), rand(N, C, T).to(dtype), rand(N, C), gen


def check(x, gate, initial, lengths, kind, coupled, g, gs):
    """All outputs and gradients of one call; x [N, C, T]"""
    leaves = [v.detach().clone().requires_grad_() for v in (x, gate, initial)]
    y, last = gatedLeak(leaves[0], leaves[1], initial=leaves[2], lengths=lengths, kind=kind, coupled=coupled, returnState=True)
    grads = torch.autograd.grad([y, last], leaves, [g, gs])
    N, C, T = x.shape
    rows = lambda v: v.reshape(N * C, -1)  # noqa: E731
    per = None if lengths is None else lengths.clamp(0, T).repeat_interleave(C)
    ref = want(rows(x), rows(gate.expand(N, C, gate.shape[-1])), initial.reshape(-1), per, kind, coupled, rows(g), gs.reshape(-1))
    assert y.dtype == x.dtype and last.dtype == torch.float32 and grads[1].dtype == gate.dtype
    close(rows(y), *ref[0])
    close(last.reshape(-1), *ref[1])
    close(rows(grads[0]), *ref[2])
    close(grads[2].reshape(-1), *ref[4])
    value, bound = (v.reshape(N, C, T) for v in ref[3])
    if gate.shape != x.shape:       # added up where the gate is broadcast: in double per neuron, else after a rounding to the type
        rounded = 0.0 if gate.shape[-1] == 1 else torch.finfo(x.dtype).eps * value.abs()
        value, bound = (v.sum_to_size(gate.shape) if v.shape != gate.shape else v for v in (value, bound + rounded + STEP * value.abs()))
        if gate.shape[-1] != 1:     # and in PyTorch's sums
            bound = bound + N * C * torch.finfo(x.dtype).eps * value.abs() + 1e-6
    close(grads[1], value, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 15, 31, 33, 64, 100, 127, 128, 129, 145, 255, 257, 300, 1000])
def test_lengths_of_rows(T, dtype):
    """Every number of lanes per row, rows that start anywhere in their 16 bytes, both kinds and inputs."""
    for kind in ('logit', 'decay'):
        for coupled in (False, True):
            x, gate, h, g, gs, _ = made(3, 23, T, dtype, kind, T + coupled)
            check(x, gate, h, None, kind, coupled, g, gs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, 14, 15, 17])
def test_many_short_rows(T, dtype):
    """Rows that end inside of vectors, more than a CTA has and not a multiple of it; with lengths, and gates per step and per row."""
    gen = torch.Generator(device="cuda").manual_seed(40 + T)
    for N, C in ((1, 127), (1, 128), (7, 43)):
        for coupled, kind in ((False, 'decay'), (True, 'logit')):
            for shape in ((N, C, T), (C, 1)):
                x, gate, h, g, gs, _ = made(N, C, T, dtype, kind, T + N, shape)
                lengths = torch.randint(-1, T + 2, (N,), device="cuda", generator=gen) if coupled else None
                check(x, gate, h, lengths, kind, coupled, g, gs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C,T", [(1, 1, 700), (1, 1, 5003), (1, 3, 20001), (2, 16, 4099), (1, 300, 2048), (1, 1500, 1030), (7, 700, 600)])
def test_long_rows_and_few(N, C, T, dtype):
    """Rows that are split among groups of lanes, and those that are just not."""
    x, gate, h, g, gs, gen = made(N, C, T, dtype, 'logit', T)
    check(x, gate, h, None, 'logit', True, g, gs)
    lengths = torch.randint(0, T + 1, (N,), device="cuda", generator=gen)
    check(x, gate, h, lengths, 'logit', False, g, gs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 1), (1, 1), (4, 1, 1), (4, 5, 1), (1, 5, 1), (4, 1, 37), (5, 37), (37,), (1,), (), (4, 5, 37)])
def test_gates_that_are_broadcast(shape, dtype):
    for lengths in (None, torch.tensor([37, 0, 12, 40], device="cuda")):
        x, gate, h, g, gs, _ = made(4, 5, 37, dtype, 'logit', 1, shape)
        check(x, gate, h, lengths, 'logit', True, g, gs)
    if len(shape) and shape[-1] == 1:           # and rows of many chunks, which are split
        x, gate, h, g, gs, _ = made(4, 5, 3001, dtype, 'decay', 2, shape)
        check(x, gate, h, None, 'decay', False, g, gs)


def test_a_gate_per_neuron_of_another_type_and_of_many_rows():
    x, _, h, g, gs, gen = made(64, 40, 200, torch.bfloat16, 'logit', 3)
    gate = torch.randn(40, 1, device="cuda", generator=gen)
    check(x, gate, h, None, 'logit', False, g, gs)
    x, _, h, g, gs, gen = made(130, 150, 9, torch.float32, 'logit', 4)
    check(x, torch.randn(1, device="cuda", generator=gen), h, None, 'logit', True, g, gs)       # one gate: 19500 rows add up
    with pytest.raises(TypeError, match="must have the type of x"):
        gatedLeak(x, torch.zeros_like(x, dtype=torch.float16))


def test_images_of_five_dimensions():
    """[N, C, H, W, T] with gates per channel, per pixel, and per sample and pixel (dimensions that do not lie together)."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 3, 4, 5, 50, device="cuda", generator=gen)
    g = torch.randn(x.shape, device="cuda", generator=gen)
    for shape in ((3, 1, 1, 1), (3, 4, 5, 1), (4, 5, 1), (2, 1, 4, 5, 1), (2, 3, 4, 5, 1), (2, 1, 1, 5, 50)):
        gate = torch.randn(shape, device="cuda", generator=gen).requires_grad_()
        (got,) = torch.autograd.grad(gatedLeak(x, gate), [gate], g)
        ref = want(x.reshape(-1, 50), gate.detach().expand(*x.shape[:-1], shape[-1]).reshape(-1, shape[-1]), None, None, 'logit', False, g.reshape(-1, 50))[3]
        value, bound = (v.reshape(x.shape).sum_to_size((1,) * (5 - len(shape)) + shape).reshape(shape) for v in (ref[0], ref[1] + 40 * STEP * ref[0].abs()))
        close(got, value, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_lies_behind_a_length_is_not_used(dtype):
    x, gate, h, g, gs, _ = made(6, 3, 333, dtype, 'logit', 6)
    lengths = torch.tensor([0, 1, 128, 332, 333, 200], device="cuda")
    clean = gatedLeak(x, gate, initial=h, lengths=lengths, returnState=True)
    behind = torch.arange(333, device="cuda") >= lengths[:, None, None]
    leaves = [torch.where(behind, float(bad), v).requires_grad_() for v, bad in ((x, "nan"), (gate, "inf"))]
    y, last = gatedLeak(*leaves, initial=h, lengths=lengths.int(), returnState=True)
    assert torch.equal(y, clean[0]) and torch.equal(last, clean[1]) and bool((y[behind.expand_as(y)] == 0).all())
    grads = torch.autograd.grad([y, last], leaves, [torch.where(behind, float("nan"), g), gs])
    for v in grads:
        assert bool((v[behind.expand_as(v)] == 0).all()) and bool(v.isfinite().all())
    assert torch.equal(last[0], h[0])
    # out of range: taken into [0, T]
    far = gatedLeak(x, gate, initial=h, lengths=lengths + torch.tensor([-5, 0, 0, 0, 7, 0], device="cuda"))
    assert torch.equal(far, clean[0])


def test_gates_at_their_ends():
    """f of 0 and 1 exactly, gates of +-infinity and of large size; a state that is not finite stays in its row and behind its step."""
    T = 300
    x = torch.ones(4, T, device="cuda")
    for gate, y in ((float("-inf"), torch.ones(T)), (float("inf"), torch.arange(1, T + 1)), (1000.0, torch.arange(1, T + 1)), (-1000.0, torch.ones(T))):
        assert torch.equal(gatedLeak(x, torch.full((1, 1), gate, device="cuda")).cpu(), y.float().expand(4, T))
        out = gatedLeak(x, torch.full_like(x, gate), coupled=True, initial=torch.full((4,), 3.0, device="cuda"))
        assert torch.equal(out.cpu(), torch.full((4, T), 3.0 if gate > 0 else 1.0))
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[1, 77] = value
        y = gatedLeak(bad, torch.full_like(x, 2.0))
        assert bool(y[[0, 2, 3]].isfinite().all()) and bool(y[1, :77].isfinite().all()) and not bool(y[1, 77:].isfinite().any())
    # a decay of zero forgets, whatever was there; negative ones alternate
    y = gatedLeak(torch.randn(2, T, device="cuda") * 1e30, torch.zeros(2, T, device="cuda"), kind='decay')
    assert bool(y.isfinite().all())
    y = gatedLeak(torch.cat([torch.ones(1, 1), torch.zeros(1, 9)], 1).cuda(), torch.full((1, 1), -0.5, device="cuda"), kind='decay')
    assert torch.equal(y.cpu(), (-0.5) ** torch.arange(10.0)[None])


@pytest.mark.parametrize("T", [1, 3, 13, 14, 15, 16, 17, 33, 101, 510, 511, 513, 1027, 8195])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("short", [False, True])
def test_rows_keep_to_themselves(T, dtype, short):
    """Rows share vectors where T is no multiple of four: what every second row and the memory around the tensors hold changes nothing elsewhere."""
    def run(other):
        rng = torch.Generator("cuda").manual_seed(T)
        leaves, R = [], 9
        for _ in range(3):
            # the tensor's first element lies on 16 bytes, its last one is followed at once by others' memory
            memory = torch.full((R * T + 64,), other, dtype=dtype, device="cuda")
            v = memory[16:16 + R * T].view(R, T)
            v.copy_(torch.randn(R, T, generator=rng, device="cuda"))
            v[1::2] = other
            leaves.append(v)
        lengths = torch.tensor([T, T, T - 1, T, 0, T, T // 2, T, T], device="cuda") if short else None
        x, gate = leaves[0].requires_grad_(), leaves[1].requires_grad_()
        y, last = gatedLeak(x, gate, lengths=lengths, returnState=True)
        return [v[::2] for v in (y, last, *torch.autograd.grad(y, [x, gate], leaves[2]))]
    clean, dirty = run(0.5), run(float("nan"))
    for a, b in zip(clean, dirty):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


def test_a_slow_leak_over_many_steps():
    """A time constant of 20000 steps over 100000: what rounding f to 32 bits would take from it is 1e-3."""
    T = 100000
    gate = torch.full((2, 1), 9.9, device="cuda")
    x = torch.ones(2, T, device="cuda")
    y = gatedLeak(x, gate)
    f = torch.sigmoid(gate[0, 0].double())
    value = (1 - f ** torch.arange(1, T + 1, device="cuda", dtype=torch.float64)) / (1 - f)
    # what is forgotten too much changes the sum by as much of itself at most; the walk: 17 times 3 steps
    close(y, value.expand(2, T), ((8 + 9.9 + 2 * 160 + 51) * STEP * value).expand(2, T))


def test_streams_of_parts_and_of_single_steps():
    x, gate, h, _, _, _ = made(3, 50, 700, torch.float32, 'logit', 8)
    whole, last = gatedLeak(x, gate, initial=h, coupled=True, returnState=True)
    value, bound = want(x.reshape(150, -1), gate.reshape(150, -1), h.reshape(-1), None, 'logit', True)[0]
    # a state is rounded to 32 bits at each part's end, and what that changes decays
    state, parts = h, []
    for a, b in ((0, 1), (1, 1), (1, 130), (130, 699), (699, 700)):
        y, state = gatedLeak(x[..., a:b], gate[..., a:b], initial=state, coupled=True, returnState=True)
        parts.append(y)
    extra = 5 * STEP * value.abs().amax(1, keepdim=True)
    close(torch.cat(parts, -1).reshape(150, -1), value, bound + extra)
    state, parts = h.clone(), []
    for t in range(200):
        parts.append(gatedLeakStep(x[..., t], gate[..., t], state, coupled=True))
    close(torch.stack(parts, -1).reshape(150, -1), value[:, :200], (bound + 200 * STEP * value.abs().amax(1, keepdim=True))[:, :200])
    assert torch.equal(parts[-1], state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,gshape", [((1,), (1,)), ((3, 7, 5), (3, 7, 5)), ((3, 7, 5), (7, 5)), ((3, 7, 5), (7, 1)), ((3, 7, 5), (3, 1, 5)), ((64, 1023), ()),
                                          ((300, 4001), (4001,)), ((0, 5), (5,)), ((2, 3), (2, 1))])
def test_single_steps(shape, gshape, dtype):
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(shape, device="cuda", generator=gen).to(dtype)
    for kind in ('logit', 'decay'):
        for gtype in {dtype, torch.float32} if gshape != shape else {dtype}:
            for coupled in (False, True):
                gate = torch.rand(gshape, device="cuda", generator=gen).to(gtype)
                state = torch.randn(shape, device="cuda", generator=gen)
                ref = want(x.reshape(-1, 1), gate.expand(shape).reshape(-1, 1), state.reshape(-1), None, kind, coupled)[0] if x.numel() else None
                version = state._version
                y = gatedLeakStep(x, gate, state, kind=kind, coupled=coupled)
                assert y.dtype == dtype and y.shape == x.shape and state._version > version
                if ref:
                    close(y.reshape(-1, 1), *ref)
                    close(state.reshape(-1, 1), *ref)


def test_gradients_against_differences():
    """d L along a direction, from central differences of the forward pass: what they leave out is four times what halving the step changes, and L
    has an error of 2^-22 of the sum of its terms."""
    x, gate, h, w, ws, gen = made(2, 9, 150, torch.float32, 'logit', 10)
    for coupled in (False, True):
        leaves = [v.clone().requires_grad_() for v in (x, gate, h)]
        grads = torch.autograd.grad(gatedLeak(*leaves[:2], initial=leaves[2], coupled=coupled, returnState=True), leaves, [w, ws])
        for i in range(3):
            v = torch.randn(leaves[i].shape, device="cuda", generator=gen)

            def L(step):
                a = [(u + step * v if k == i else u) for k, u in enumerate((x, gate, h))]
                y, s = gatedLeak(*a[:2], initial=a[2], coupled=coupled, returnState=True)
                return (y.double() * w).sum() + (s.double() * ws).sum(), 2.0 ** -22 * ((y.double() * w).abs().sum() + (s.double() * ws).abs().sum())
            d = {}
            for step in (2.0 ** -5, 2.0 ** -6):
                (a, ea), (b, eb) = L(step), L(-step)
                d[step] = ((a - b) / (2 * step), (ea + eb) / (2 * step))
            (a, ea), (b, eb) = d.values()
            assert abs((grads[i].double() * v).sum() - b) <= 4 * abs(a - b) + 5 * ea + 5 * eb


def test_strides_offsets_and_expanded_gradients():
    x, gate, h, g, _, _ = made(4, 6, 100, torch.float32, 'logit', 11)
    y = gatedLeak(x, gate, initial=h)
    assert torch.equal(gatedLeak(x.transpose(0, 2).contiguous().transpose(0, 2), gate, initial=h.t().contiguous().t()), y)
    store = torch.zeros(x.numel() + 8, device="cuda")
    for off in (1, 2, 3):       # tensors that start off 16 bytes: their steps are loaded one by one
        moved = store[off:off + x.numel()].view(x.shape)
        moved.copy_(x)
        assert torch.equal(gatedLeak(moved, gate, initial=h), y)
    leaf = x.clone().requires_grad_()
    (a,) = torch.autograd.grad(gatedLeak(leaf, gate, initial=h).sum(), [leaf])
    (b,) = torch.autograd.grad(gatedLeak(leaf, gate, initial=h), [leaf], torch.ones_like(x))
    assert torch.equal(a, b)
    # only one of the outputs, only one of the inputs
    gl = gate.clone().requires_grad_()
    last = gatedLeak(x, gl, initial=h, returnState=True)[1]
    (c,) = torch.autograd.grad(last.sum(), [gl])
    ref = want(x.reshape(24, -1), gate.reshape(24, -1), h.reshape(-1), None, 'logit', False, torch.zeros(24, 100, device="cuda"),
               torch.ones(24, device="cuda"))[3]
    close(c.reshape(24, -1), *ref)


def test_empty_tensors():
    for shape, gshape in (((0, 5, 7), (0, 5, 7)), ((2, 0, 7), (2, 0, 7)), ((3, 0, 7), (3, 1, 1)), ((2, 3, 0), (2, 3, 0)), ((2, 3, 0), (3, 1)), ((0, 3, 4), (3, 1))):
        x, gate = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(gshape, device="cuda", requires_grad=True)
        h = torch.ones(shape[:-1], device="cuda", requires_grad=True)
        y, s = gatedLeak(x, gate, initial=h, returnState=True)
        assert y.shape == x.shape and torch.equal(s, h)
        grads = torch.autograd.grad([y, s], [x, gate, h], [torch.ones_like(y), torch.ones_like(s)])
        assert bool((grads[1] == 0).all()) and torch.equal(grads[2], torch.ones_like(h))


def test_graph_capture_and_streams():
    """A captured training step replays with new contents, and a call on another stream gives the same bits."""
    x, gate, h, g, gs, _ = made(2, 3, 9001, torch.float32, 'logit', 12)
    leaves = [v.requires_grad_() for v in (x, gate, h)]

    def step():
        y, s = gatedLeak(*leaves[:2], initial=leaves[2], returnState=True)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [g, gs])]
    eager = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(-1.0), h.mul_(-1.0)
    graph.replay()
    assert torch.equal(out[0], -eager[0]) and torch.equal(out[2], eager[2]) and torch.equal(out[3], -eager[3])


def test_second_derivatives_are_refused():
    x, gate, h, g, _, _ = made(1, 2, 10, torch.float32, 'logit', 13)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(gatedLeak(x, gate), [x], g, create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        dx.sum().backward()


def test_refusals():
    x, gate, h, _, _, _ = made(2, 3, 10, torch.float32, 'logit', 14)
    bad = torch.zeros(2, 3, 9, device="cuda")
    for call in (lambda: gatedLeak(x, bad), lambda: gatedLeak(x, gate[None]), lambda: gatedLeak(x, gate, initial=h[0]),
                 lambda: gatedLeak(x, gate, lengths=torch.zeros(3, dtype=torch.long, device="cuda")), lambda: gatedLeak(x, gate, kind='other'),
                 lambda: gatedLeakStep(x[..., 0], gate[..., 0], h[0]), lambda: gatedLeakStep(x[..., 0].requires_grad_(), gate[..., 0], h),
                 lambda: gatedLeakStep(x[..., 0], gate[..., 0], h.t().contiguous().t())):
        with pytest.raises(ValueError):
            call()
    x = x.detach()
    for call in (lambda: gatedLeak(x, gate, lengths=torch.zeros(2, device="cuda")), lambda: gatedLeakStep(x[..., 0], gate[..., 0], h.double())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: gatedLeak(x, gate.cpu()), lambda: gatedLeak(x.double(), gate), lambda: gatedLeak(x, gate, initial=h.cpu()),
                 lambda: gatedLeak(x, gate, lengths=torch.zeros(2, dtype=torch.long))):
        with pytest.raises(RuntimeError):
            call()


def test_layer_of_learnable_leaks():
    """spikeLayer.leak per neuron and per channel, its single steps, and gatedPsp."""
    neuron = {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1}
    net = layer.spikeLayer(neuron, {"Ts": 1.0, "tSample": 60}).cuda()
    x = torch.randn(2, 6, 1, 1, 60, device="cuda")
    leak = net.leak(6, coupled=True).cuda()
    assert leak.gate.shape == (6, 1, 1, 1) and 0.5 <= float(torch.sigmoid(leak.gate).min()) and float(torch.sigmoid(leak.gate).max()) <= 0.9901
    y = leak(x)
    assert torch.equal(y, net.gatedPsp(x, leak.gate, coupled=True))
    y.sum().backward()
    assert leak.gate.grad.shape == leak.gate.shape
    state, steps = torch.zeros(2, 6, 1, 1, device="cuda"), []
    for t in range(60):
        steps.append(leak.step(x[..., t], state))
    assert torch.allclose(torch.stack(steps, -1), y, rtol=0, atol=60 * STEP * float(y.abs().max()))
    assert net.leak((4, 5, 3)).gate.shape == (4, 5, 3, 1)
    with pytest.raises(Exception, match="inputSize"):
        net.leak((4, 5))
