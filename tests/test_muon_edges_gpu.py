"""GPU: the orthogonalised updates at their edges - refused calls, a first step in a capture, every way of sharing out the tiles."""
import math

import pytest
import torch

from slayerpytorch_b200 import optim
from tests.test_muon_gpu import TYPES, gradient, near, slack, step_case, want_orthogonal, want_step

pytestmark = pytest.mark.gpu


def test_a_first_step_of_the_optimiser_is_not_captured():
    """Its momenta would be made, and set to zero, by every replay."""
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((20, 30), (8, 4, 3, 3))]
    for p in params:
        p.grad = torch.randn_like(p)
    before = [p.detach().clone() for p in params]
    opt = optim.Muon(params)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(params, before)) and not any("momentum" in opt.state[p] for p in params)
    # after a step outside, replays are steps
    other = [torch.nn.Parameter(b.clone()) for b in before]
    eager = optim.Muon(other)
    for q, p in zip(other, params):
        q.grad = p.grad
    for _ in range(4):
        eager.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(params, other):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["momentum"], eager.state[q]["momentum"])


def test_a_refused_step_changes_nothing():
    """Lists of several types are worked on one type after the other: what the second is refused for is found before the first."""
    ws, gs, ms = step_case([(24, 30), (16, 20)], torch.float32, 11)
    w, g, m = ([t.cuda() for t in ts] for ts in (ws, gs, ms))
    long = torch.zeros(1, (1 << 22) + 1, device="cuda")       # longer than a matrix may be
    far = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16)
    for second in ((w[1].double(), g[1].double(), m[1]), (w[1].bfloat16(), g[1], m[1]), (w[1].bfloat16(), g[1].bfloat16(), m[1].bfloat16()),
                   (w[1].bfloat16(), g[1].bfloat16(), m[1][:8]), (w[1].bfloat16(), g[1].bfloat16()[:8], m[1]), (w[1].cpu(), g[1].cpu(), m[1].cpu()),
                   (w[1].bfloat16(), g[1].bfloat16().cpu(), m[1]), (far.expand(16, 20), g[1].bfloat16(), m[1]),
                   (long.bfloat16(), long.bfloat16(), long.clone())):
        with pytest.raises((RuntimeError, ValueError)):
            optim.muonStep([w[0], second[0]], [g[0], second[1]], [m[0], second[2]], lr=0.1)
        assert torch.equal(w[0].cpu(), ws[0]) and torch.equal(m[0].cpu(), ms[0])
    for more in (dict(steps=0), dict(eps=-1.0), dict(coefficients=(9.0, 0.0, 0.0))):
        with pytest.raises(RuntimeError):
            optim.muonStep(w, g, m, lr=0.1, **more)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(w + m, ws + ms))


def blocks(v):
    return (v + 127) // 128


def sharing(shapes, dtype):
    """How a launch of matrices that do not stay on the chip shares out its tiles, and how many tiles there are for each CTA (pair)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    sides = [(min(s), max(s)) for s in shapes]
    pairs = sum(((blocks(m) + 1) // 2) * ((blocks(n) + 1) // 2) for m, n in sides)
    if pairs >= sms // 2:
        return "pairs", pairs / (sms // 2)
    if sum(blocks(m) * (blocks(m) + 1) // 2 for m, _ in sides) * 4 <= sms:
        return "shared", 1
    return "alone", sum(blocks(m) * blocks(n) for m, n in sides) / sms


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1100, 1300), (1300, 1100), (4, 512, 512), (4, 513, 600), (2, 768, 777), (1664, 1280), (30, 200, 140)])
def test_orthogonalize_tiles_of_a_cta_alone(shape, dtype):
    assert sharing([shape[-2:]] * math.prod(shape[:-2]), dtype)[0] == "alone"
    x = gradient(shape, sum(shape), dtype)
    near(optim.orthogonalize(x.cuda()), want_orthogonal(x.cuda()).cpu(), dtype, min(shape[-2:]) * math.prod(shape[:-2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [[(1100, 1300)], [(512, 600), (640, 512), (30, 20), (10, 512), (700, 800)]])
def test_muon_step_tiles_of_a_cta_alone(shapes, dtype):
    assert sharing(shapes, dtype)[0] == "alone"
    check_step(shapes, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [[(2600, 7700)], [(300, 520)] * 17 + [(1290, 5000)] * 3 + [(5000, 1290), (4, 9)]])
def test_more_tiles_than_are_worked_out_ahead(shapes, dtype):
    """A CTA's first four tiles are located once, later ones as they come."""
    mode, each = sharing(shapes, dtype)
    assert mode == "pairs" and each > 4
    check_step(shapes, dtype)


def check_step(shapes, dtype):
    ws, gs, ms = ([t.cuda() for t in ts] for ts in step_case(shapes, dtype, 60))
    dw, dm = [t.clone() for t in ws], [t.clone() for t in ms]
    optim.muonStep(dw, gs, dm, lr=0.03, weightDecay=0.1)
    for w, g, m, gw, gm in zip(ws, gs, ms, dw, dm):
        want, mom, step = want_step(w, g, m, 0.03, decay=0.1)
        assert bool(((gm.double() - mom).abs() <= 2.0 ** -23 * (m.double().abs() + mom.abs())).all())
        off = torch.linalg.vector_norm(gw.double() - want)
        rank = min(w.shape)
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -22
        assert float(off) <= step * slack(dtype, rank) * math.sqrt(rank) * 1.2 + half * float(torch.linalg.vector_norm(want)) + 1e-30


def off(got, want):
    return float(torch.linalg.vector_norm(got.double() - want) / torch.linalg.vector_norm(want))


def fp32_products(x):
    """The definition in fp32 throughout."""
    a, b, c = optim.COEFFICIENTS
    if x.shape[0] > x.shape[1]:
        return fp32_products(x.mT).mT
    x = x / (torch.linalg.vector_norm(x) + 1e-7)
    for _ in range(5):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


@pytest.mark.parametrize("strong", [True, False])
@pytest.mark.parametrize("shape", [(16, 50), (64, 288), (100, 300), (128, 128), (128, 256), (128, 512), (128, 1024), (128, 2500), (10, 4096),
                                   (200, 256), (333, 2000), (2000, 333), (512, 2312), (700, 700), (1100, 1300), (2048, 2048)])
def test_errors_against_those_of_fp32_products(shape, strong):
    """Products of two 16-bit parts (22 bits) whose sums beyond 64 to 192 products are added up in fp32 are no further off than fp32
    products.  In matrices that stay on the chip (up to 128 rows) fp32's sums are short, 128 roundings to either side of about
    sqrt(128 / 12) = 3.3 half steps; a sum of 64 products in tensor memory has 4 large additions that are cut by half a step of what
    is there, (1 + 2 + 3 + 4) / 4 = 2.5 half steps to one side, and two such sums are added up; the parts are rounded 1.5 times as
    coarsely as fp32 values.  2.5 sqrt(1 + 1.5^2) against 3.3 sqrt(1 + 1): less than twice as far off where all of it points one way."""
    x = (gradient(shape, 5) if strong else torch.randn(shape, generator=torch.Generator().manual_seed(5))).cuda()
    want = want_orthogonal(x)
    assert not torch.backends.cuda.matmul.allow_tf32
    assert off(optim.orthogonalize(x), want) <= (2 if min(shape) <= 128 else 1) * off(fp32_products(x), want)


@pytest.mark.parametrize("strong", [True, False])
@pytest.mark.parametrize("shape", [(4, 30), (16, 50), (32, 144), (64, 288), (100, 300), (128, 1024), (10, 4096), (4096, 10), (333, 2000), (700, 700),
                                   (1100, 1300), (1023, 2049), (2048, 2048), (3, 30000), (300, 9000)])
def test_errors_of_bfloat16_matrices_are_their_rounding(shape, strong):
    """Products of 22 bits leave nothing to be seen beside the result's rounding to 8 bits: `slack` of float32 matrices, and the bias of sums of
    1024 products in tensor memory (192 additions that are cut by half a step each, 2^-24 of the sum, and multiplied by at most 1.71 in each
    later step: 1 + 1.71 + ... + 1.71^4 = 18.9)."""
    x = (gradient(shape, 6) if strong else torch.randn(shape, generator=torch.Generator().manual_seed(6))).bfloat16().cuda()
    want = want_orthogonal(x)
    assert off(optim.orthogonalize(x), want) <= math.hypot(off(want.bfloat16(), want), slack(torch.float32, min(shape)) + 192 * 2.0 ** -24 * 18.9)


def test_stacks_and_lists_that_a_launch_does_not_hold():
    """More matrices than 4 GB of workspace take at once; each comes out as it does alone."""
    x = torch.randn(40, 4096, 4096, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16)
    got = optim.orthogonalize(x)
    for i in (0, 29, 30, 31, 32, 39):
        assert torch.equal(got[i], optim.orthogonalize(x[i]))
    small = torch.randn(30, 300, 500, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda", dtype=torch.bfloat16)
    grads = [t for pair in zip(x, small) for t in pair] + list(x[30:])
    weights, momenta = [torch.zeros_like(g) for g in grads], [torch.zeros(g.shape, device="cuda") for g in grads]
    optim.muonStep(weights, grads, momenta, lr=1.0, nesterov=False, adjust=None)
    for w, g, m in zip(weights, grads, momenta):
        assert torch.equal(m, g.float())
    for i in (0, 28, 58, 59, 60, 69):
        if grads[i].shape[0] == 4096:
            assert torch.equal(weights[i], -optim.orthogonalize(grads[i]))
        else:
            near(-weights[i], want_orthogonal(grads[i]).cpu(), torch.bfloat16, 300)
