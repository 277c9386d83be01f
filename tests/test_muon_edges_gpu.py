"""GPU: the orthogonalised updates at their edges - refused calls, a first step in a capture, every way of sharing out the tiles."""

import pytest
import torch

from slayerpytorch_b200 import optim
from tests.test_muon_gpu import step_case

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
