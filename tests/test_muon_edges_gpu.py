"""GPU: the orthogonalised updates at their edges - refused calls, a first step in a capture, every way of sharing out the tiles."""

import pytest
import torch

from slayerpytorch_b200 import optim

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
