"""GPU: orthogonalised updates against their definition in 64 bits.

Tolerances (relative to the root mean square of the result, and to its norm).  Each step multiplies a perturbation of X in the
direction of a singular value s by at most p(s)/s <= 3.4445 for small s, so a relative rounding e of X0 grows to 3.4445^5 e = 485 e in
the weakest directions; of X0 as a whole it grows by |X5|_F / |X0|_F = |X5|_F, since |X0|_F is one.  With t roundings of one step
(x, a, b and the sums) the norm of the error relative to that of the result is below 485 t e / sqrt(rank) plus 5 t e for the
directions that have arrived (|p'| <= 4 there, which random signs and five steps keep near t e * 4^2).  float32 / float16 inputs:
products of 22 bits with fp32 sums, e = 2^-22, t = 8; bfloat16: products of fp16 values, e = 2^-12, t = 4.  The result's own
rounding is half a step of its type."""
import math
import os
import subprocess
import sys

import pytest
import torch

from slayerpytorch_b200 import layer, loss, optim

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
A, B, C = optim.COEFFICIENTS


def want_orthogonal(x, steps=5, coef=(A, B, C), eps=1e-7):
    a, b, c = coef
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * g @ g) @ x
    return x.mT if tall else x


def slack(dtype, rank, steps=5, slope=A):
    e, t = (2.0 ** -12, 4) if dtype == torch.bfloat16 else (2.0 ** -22, 8)
    return slope ** steps * t * e / math.sqrt(max(1, rank)) + 16 * t * e


def near(got, want, dtype, rank, work=None):
    """work: the type whose products were used"""
    assert got.shape == want.shape
    off = torch.linalg.vector_norm(got.double().cpu() - want)
    norm = float(torch.linalg.vector_norm(want))
    bound = (slack(work or dtype, rank) + torch.finfo(dtype).eps / 2) * norm + 1e-30
    assert float(off) <= bound, "off by %g of %g" % (float(off) / max(norm, 1e-30), bound / max(norm, 1e-30))


def gradient(shape, seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r, c = shape[-2], shape[-1]
    k = min(4, r, c)
    low = torch.randn(*shape[:-1], k, generator=gen) @ torch.randn(*shape[:-2], k, c, generator=gen)
    return ((low + torch.randn(shape, generator=gen)) * 1e-3).to(dtype)


SIZES = [(1, 1), (1, 7), (5, 1), (2, 3), (16, 50), (32, 144), (64, 288), (10, 4096), (127, 129), (128, 128), (129, 127), (200, 256), (257, 300),
         (130, 1000), (700, 65), (128, 2500), (128, 2600), (100, 5000), (64, 6200), (8100, 24), (17, 8192), (33, 65), (113, 300), (512, 600), (300, 2100), (1030, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SIZES)
def test_orthogonalize(shape, dtype):
    x = gradient(shape, sum(shape), dtype)
    got = optim.orthogonalize(x.cuda())
    assert got.dtype == dtype
    near(got, want_orthogonal(x), dtype, min(shape))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1500, 3300), (2310, 2050), (10, 400, 900), (9, 1, 640, 513), (40, 300, 150)])
def test_orthogonalize_many_tiles(shape, dtype):
    """Enough tiles for pairs of CTAs, row and column blocks that have no partner, more tiles than CTAs."""
    x = gradient(shape, sum(shape), dtype)
    near(optim.orthogonalize(x.cuda()), want_orthogonal(x.cuda()).cpu(), dtype, min(shape[-2:]) * math.prod(shape[:-2]))


@pytest.mark.parametrize("dtype", TYPES)
def test_orthogonalize_stacks_orders_and_scales(dtype):
    x = gradient((2, 3, 40, 70), 5, dtype)
    want = want_orthogonal(x)
    d = x.cuda()
    got = optim.orthogonalize(d)
    near(got, want, dtype, 40)
    near(optim.orthogonalize(d.mT).mT, want, dtype, 40)
    near(optim.orthogonalize(d[:, 1:]), want[:, 1:], dtype, 40)
    assert torch.equal(optim.orthogonalize(d[1, 2]), got[1, 2])             # a matrix does not depend on its neighbours
    many = gradient((130, 9, 20), 6, dtype)
    near(optim.orthogonalize(many.cuda()), want_orthogonal(many), dtype, 9)
    if dtype != torch.float16:                                              # 1e30, and its square past the largest float32
        for scale in (1e30, 1e-30):
            y = (gradient((40, 70), 5) * scale).to(dtype)
            near(optim.orthogonalize(y.cuda(), eps=0.0), want_orthogonal(y, eps=0.0), dtype, 40)
    big = torch.randn(60, 61, generator=torch.Generator().manual_seed(1)).to(dtype)
    for coef, steps in (((1.5, -0.5, 0.0), 12), ((15 / 8, -10 / 8, 3 / 8), 1), ((2.0, -1.5, 0.5), 20)):
        got = optim.orthogonalize(big.cuda(), steps=steps, coefficients=coef)
        want = want_orthogonal(big, steps, coef)
        off = float(torch.linalg.vector_norm(got.double().cpu() - want) / torch.linalg.vector_norm(want))
        # the weakest direction grows by at most sqrt(60) / its size before it arrives, and slopes are below 1 from there
        assert off <= slack(dtype, 1, 0) * 60 + torch.finfo(dtype).eps / 2


def test_orthogonalize_degenerate_matrices():
    dev = "cuda"
    assert bool((optim.orthogonalize(torch.zeros(3, 20, 30, device=dev)) == 0).all())
    assert optim.orthogonalize(torch.zeros(0, 20, 30, device=dev)).shape == (0, 20, 30)
    assert optim.orthogonalize(torch.zeros(2, 0, 30, device=dev)).shape == (2, 0, 30)
    for bad in (float("nan"), float("inf")):
        x = gradient((3, 50, 200), 9)
        x[1, 7, 100] = bad
        got = optim.orthogonalize(x.cuda()).cpu()
        assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[[0, 2]]).all())
        near(got[[0, 2]], want_orthogonal(x[[0, 2]]), torch.float32, 50)
    # one strong direction and nothing else: the noise of 24 bits is what the others consist of
    u, v = torch.randn(50, 1, dtype=torch.float64), torch.randn(1, 90, dtype=torch.float64)
    x = (u @ v).float()
    got = optim.orthogonalize(x.cuda()).double().cpu()
    strong = float((u / u.norm()).T @ got @ (v / v.norm()).T)
    s = 1.0
    for _ in range(5):
        s = A * s + B * s ** 3 + C * s ** 5
    assert abs(strong - s) < 1e-4
    assert float(torch.linalg.vector_norm(got)) < s + 485 * 8 * 2.0 ** -22


@pytest.mark.parametrize("shape", [(20, 30), (30, 20), (200, 260)])
def test_orthogonalize_of_the_smallest_numbers(shape):
    """A norm whose inverse is no float: with eps = 0 the result is that of the same matrix scaled by a power of two, bit for bit."""
    x = torch.randint(-3, 4, shape, generator=torch.Generator().manual_seed(2)).float().cuda()
    tiny = torch.ldexp(torch.ldexp(x, torch.tensor(-100.0, device="cuda")), torch.tensor(-49.0, device="cuda"))
    assert float(tiny.double().abs().max()) == 3 * 2.0 ** -149
    assert torch.equal(optim.orthogonalize(tiny, eps=0.0), optim.orthogonalize(x, eps=0.0))


def test_the_first_call_of_a_process_in_a_graph():
    code = '''
import torch
from slayerpytorch_b200 import optim
x = [torch.randn(s, device="cuda") for s in ((300, 500), (20, 30))]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = [optim.orthogonalize(v) for v in x]
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, optim.orthogonalize(b)) for a, b in zip(y, x))
print("as eager")
'''
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0 and "as eager" in done.stdout, done.stderr[-2000:]


def test_two_streams_at_once():
    xs = [torch.randn(700, 900, device="cuda"), torch.randn(60, 400, device="cuda"), torch.randn(1100, 1300, device="cuda")]
    want = [optim.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(5):
        for x, st, g in zip(xs, streams, got):
            with torch.cuda.stream(st):
                g.append(optim.orthogonalize(x))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


def test_orthogonalize_is_repeatable_and_stream_ordered():
    x = gradient((300, 500), 3).cuda()
    first = optim.orthogonalize(x)
    for _ in range(3):
        assert torch.equal(optim.orthogonalize(x), first)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(optim.orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, first) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = optim.orthogonalize(x)
    x.copy_(gradient((300, 500), 4))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, optim.orthogonalize(x))


# -------------------------------------------------------------------------------------------------- a step
def want_step(w, g, m, lr, mu=0.95, nesterov=True, decay=0.0, adjust="shape"):
    g, m = g.double(), m.double()
    m = mu * m + g
    u = (g + mu * m if nesterov else m).flatten(1)
    r, c = u.shape
    factor = {"shape": math.sqrt(max(1.0, r / c)), "rms": 0.2 * math.sqrt(max(r, c)), None: 1.0}[adjust]
    return w.double() * (1 - lr * decay) - lr * factor * want_orthogonal(u).reshape(w.shape), m, lr * factor


def step_case(shapes, dtype, seed):
    ws, gs, ms = [], [], []
    for i, s in enumerate(shapes):
        flat = (s[0], math.prod(s[1:]))
        ws.append((torch.randn(s, generator=torch.Generator().manual_seed(seed + i)) / math.sqrt(flat[1])).to(dtype))
        gs.append(gradient(flat, seed + 100 + i, dtype).reshape(s))
        ms.append(gradient(flat, seed + 200 + i).reshape(s) * 5)
    return ws, gs, ms


CNN = [(16, 2, 5, 5, 1), (32, 16, 3, 3, 1), (64, 32, 3, 3, 1), (10, 64, 8, 8, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [CNN, [(512, 2312, 1, 1, 1), (10, 512, 1, 1, 1)], [(256, 200), (200, 256), (1, 1), (1, 500), (77, 1)],
                                    [(12, 30 + i) for i in range(101)]])
@pytest.mark.parametrize("nesterov,decay,adjust", [(True, 0.0, "shape"), (False, 0.3, "rms"), (True, 0.1, None)])
def test_muon_step(shapes, dtype, nesterov, decay, adjust):
    ws, gs, ms = step_case(shapes, dtype, 40)
    dw, dg, dm = ([t.cuda() for t in ts] for ts in (ws, gs, ms))
    optim.muonStep(dw, dg, dm, lr=0.03, nesterov=nesterov, weightDecay=decay, adjust=adjust)
    for w, g, m, gw, gm, g0 in zip(ws, gs, ms, dw, dm, dg):
        want, mom, step = want_step(w, g, m, 0.03, nesterov=nesterov, decay=decay, adjust=adjust)
        # mu itself is rounded to fp32, then the product and the sum
        assert bool(((gm.double().cpu() - mom).abs() <= 2.0 ** -23 * (m.double().abs() + mom.abs())).all())
        assert torch.equal(g0.cpu(), g)
        off = torch.linalg.vector_norm(gw.double().cpu() - want)
        rank = min(w.shape[0], w.numel() // w.shape[0])
        norm = math.sqrt(rank) * 1.2
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -22
        assert float(off) <= step * slack(dtype, rank) * norm + half * float(torch.linalg.vector_norm(want)) + 1e-30


def test_muon_step_weights_in_other_orders_and_of_mixed_types():
    ws, gs, ms = step_case([(24, 6, 3, 3), (24, 6, 3, 3), (30, 20)], torch.float32, 7)
    plain = [t.cuda() for t in ws]
    optim.muonStep(plain, [t.cuda() for t in gs], [t.cuda() for t in ms], lr=0.1)
    last = ws[0].cuda().to(memory_format=torch.channels_last)
    turned = ws[2].t().contiguous().cuda().t()
    half = ws[1].cuda().bfloat16()
    version = last._version
    optim.muonStep([last, half, turned], [gs[0].cuda().to(memory_format=torch.channels_last), gs[1].cuda().bfloat16(), gs[2].cuda()],
                   [t.cuda() for t in ms], lr=0.1)
    assert torch.equal(last, plain[0]) and torch.equal(turned, plain[2]) and last._version > version
    want, _, _ = want_step(ws[1].bfloat16(), gs[1].bfloat16(), ms[1], 0.1)
    assert float((half.double().cpu() - want).abs().max()) < 0.01


def test_muon_optimiser_matches_the_function_and_keeps_its_state():
    ws, gs, ms = step_case([(40, 30), (20, 5, 3, 3, 1)], torch.bfloat16, 3)
    params = [torch.nn.Parameter(w.cuda()) for w in ws]
    opt = optim.Muon(params, lr=0.05, weightDecay=0.2)
    mine, moms = [w.cuda() for w in ws], [torch.zeros_like(w, dtype=torch.float32).cuda() for w in ws]
    for k in range(3):
        grads = [(g * (k + 1)).cuda() for g in gs]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        optim.muonStep(mine, grads, moms, lr=0.05, weightDecay=0.2)
    for p, w, m in zip(params, mine, moms):
        assert torch.equal(p.detach(), w) and torch.equal(opt.state[p]["momentum"], m)
    again = optim.Muon([torch.nn.Parameter(p.detach().clone()) for p in params])
    again.load_state_dict(opt.state_dict())
    for p, m in zip(again.param_groups[0]["params"], moms):
        kept = again.state[p]["momentum"]
        assert kept.dtype == torch.float32 and torch.equal(kept, m) and kept.data_ptr() != m.data_ptr()
    # parameters without a gradient stay as they are; a closure's loss comes back
    params[0].grad = None
    before = params[0].detach().clone()
    assert opt.step(lambda: 3.0) == 3.0 and torch.equal(params[0].detach(), before)


def test_muon_step_in_a_graph():
    ws, gs, ms = step_case(CNN, torch.float32, 9)
    a = [[t.cuda() for t in ts] for ts in (ws, gs, ms)]
    b = [[t.cuda() for t in ts] for ts in (ws, gs, ms)]
    for _ in range(3):
        optim.muonStep(*a, lr=0.02)
    side = [[t.clone() for t in ts] for ts in b]
    optim.muonStep(*side, lr=0.02)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.muonStep(*b, lr=0.02)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(a[0] + a[2], b[0] + b[2]):
        assert torch.equal(x, y)


def test_a_spiking_network_trained_by_reward_with_muon():
    """Layers, choices, their loss and its gradient, and the update of the weights, run together."""
    d = {"neuron": {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1},
         "simulation": {"Ts": 1.0, "tSample": 60},
         "training": {"error": {"type": "Policy", "tgtSpikeRegion": {"start": 0, "stop": 60}, "countScale": 0.2, "clip": 0.2, "klCoef": 0.01}}}
    torch.manual_seed(5)
    net = layer.spikeLayer(d["neuron"], d["simulation"]).cuda()
    first, second = net.dense(30, 40).cuda(), net.dense(40, 6).cuda()
    error = loss.spikeLoss(d).cuda()
    opt = optim.Muon(list(first.parameters()) + list(second.parameters()), lr=0.05)
    x = (torch.rand(24, 30, 1, 1, 60, device="cuda") < 0.2).float()
    good = torch.randint(0, 6, (24,), device="cuda")
    ref = None
    for _ in range(4):
        out = net.spike(second(net.psp(net.spike(first(net.psp(x))))))
        with torch.no_grad():
            counts = out.sum(-1).reshape(24, 6) * 0.2
            choice = torch.multinomial(torch.softmax(counts, 1), 1)[:, 0]
            old = error.actionLogProb(out, choice)
            ref = old if ref is None else ref
        value = error.policy(out, choice, old, (choice == good).float() - 0.5, refLogProb=old - 0.1)
        opt.zero_grad()
        value.backward()
        before = [p.detach().clone() for p in opt.param_groups[0]["params"]]
        opt.step()
        for p, b in zip(opt.param_groups[0]["params"], before):
            moved = torch.linalg.vector_norm((p.detach() - b).flatten(1).double(), 2)
            r, c = p.shape[0], p.numel() // p.shape[0]
            assert bool(torch.isfinite(p).all())
            assert float(moved) <= 0.05 * math.sqrt(max(1, r / c)) * math.sqrt(min(r, c)) * 1.25


def test_muon_refusals_on_the_device():
    w, g, m = torch.zeros(4, 5, device="cuda"), torch.zeros(4, 5, device="cuda"), torch.zeros(4, 5, device="cuda")
    for bad in ([w], [g.bfloat16()], [m]), ([w], [g[:3]], [m]), ([w], [g], [m.bfloat16()]), ([w.double()], [g.double()], [m]), ([w], [g.cpu()], [m]):
        with pytest.raises(RuntimeError):
            optim.muonStep(*bad, lr=0.1)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        optim.orthogonalize(w.double())
    with pytest.raises(RuntimeError, match="grow past"):
        optim.orthogonalize(w, coefficients=(10.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="steps"):
        optim.orthogonalize(w, steps=0)
    with pytest.raises(RuntimeError, match="a matrix of"):
        optim.orthogonalize(torch.zeros(1, 1, device="cuda").expand(33000, 33000))
