"""GPU: what layers keep in 8 bits, when they do, and what comes back at the ends of a type."""
import pytest
import torch

from slayerpytorch_b200 import checkpoint, layer

pytestmark = pytest.mark.gpu

NEURON = {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1}


@pytest.mark.parametrize("T", [32, 33, 64, 100])
def test_the_largest_float16_values_come_back_finite(T):
    """Values above 65024 are kept as 64 * 2^10, which is no float16: they come back as the largest one, off by less than half a step of 2^10."""
    most = torch.finfo(torch.float16).max
    values = torch.cat([torch.arange(64992, 65505, 32), torch.tensor([1.0, 700.0, 1e4, 6e4])])
    x = values[torch.randint(0, len(values), (50, T), generator=torch.Generator().manual_seed(T))].half()
    x[:, ::32] = most
    x[::2] *= -1
    x = x.cuda()
    kept = checkpoint.compress(x)
    exact, got = kept.restore(torch.float32), kept.restore()
    assert got.dtype == torch.float16 and bool(got.isfinite().all())
    assert torch.equal(got.float(), exact.clamp(-most, most)) and float(exact.max()) == 65536
    assert bool(((got.float() - x.float()).abs() <= most / 127).all())
    # a float32 tensor in float16: rounded to it, infinities where it is beyond
    far = checkpoint.compress(torch.full((1, T), 3e5, device="cuda"))
    assert bool(far.restore(torch.float16).isposinf().all()) and bool(far.restore().isfinite().all())


def test_layers_keep_nothing_without_gradients(monkeypatch):
    """In evaluation a layer that keeps 8 bits does what the plain one does."""
    net = layer.spikeLayer(NEURON, {"Ts": 1.0, "tSample": 90}).cuda()
    dense, plain = net.dense(20, 11, checkpoint=True).cuda(), net.dense(20, 11).cuda()
    plain.load_state_dict(dense.state_dict())
    x = torch.rand(3, 20, 1, 1, 90, device="cuda")
    u = 8.0 * torch.randn(3, 11, 1, 1, 90, device="cuda")
    spikes = net.spike(u.clone())

    def refuse(x):
        raise AssertionError("compressed without need")
    monkeypatch.setattr(layer.slayerCuda, "compress8", refuse)
    leaf = u.clone().requires_grad_()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            assert torch.equal(dense(x), plain(x))
    with torch.no_grad():
        assert torch.equal(net.spike(leaf, checkpoint=True), spikes)
    with pytest.raises(AssertionError, match="without need"):
        dense(x)


def test_memory_between_the_passes():
    """A dense layer and its neurons hold 33/128 of what they hold without checkpoints, beside the spikes."""
    net = layer.spikeLayer(NEURON, {"Ts": 1.0, "tSample": 320}).cuda()
    N, I, O, T = 16, 700, 500, 320
    x = (torch.rand(N, I, 1, 1, T, device="cuda") < 0.1).float()
    held = {}
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731  (blocks are up to 1 MB larger than what is asked for)
    for keep in (False, True):
        dense = net.dense(I, O, checkpoint=keep).cuda()
        for _ in range(2):          # the first one may make libraries' workspaces
            torch.cuda.synchronize()
            before = asked()
            s = net.spike(dense(net.psp(x)), checkpoint=keep)
            held[keep] = asked() - before - s.numel() * 4
            s.sum().backward()
            del s
            dense.weight.grad = None
    both = N * (I + O) * T * 4
    assert both <= held[False] <= both + 65536
    assert both * 33 // 128 <= held[True] <= both * 33 // 128 + 65536


def test_a_replayed_network_of_them():
    """All of a captured training step's results, the gradient of the leak's gates among them, are the eager step's."""
    torch.manual_seed(4)
    net = layer.spikeLayer(NEURON, {"Ts": 1.0, "tSample": 500}).cuda()
    fc1, leak, fc2 = net.dense(40, 60, checkpoint=True).cuda(), net.leak(60).cuda(), net.dense(60, 10, checkpoint=True).cuda()
    x = (torch.rand(4, 40, 1, 1, 500, device="cuda") < 0.1).float()
    weights = [fc1.weight, leak.gate, fc2.weight]

    def step():
        s = net.spike(leak(fc1(net.psp(x))), checkpoint=True)
        out = net.spike(fc2(net.psp(s)), checkpoint=True)
        return [out, *torch.autograd.grad(out.sum(), weights)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    eager = [v.detach().clone() for v in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        for v in out:
            v.detach().zero_()
        graph.replay()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("power", [-60, -110, -120, -130, -145])
def test_weight_gradients_of_tiny_gradients(power):
    """A gradient's three bfloat16 parts leave out less than 2^-133 of it; K = 256 products of float32 precision beside that (test_checkpoint_gpu.py)."""
    gen = torch.Generator(device="cuda").manual_seed(-power)
    x = torch.randint(-127, 128, (4, 30, 1, 1, 64), device="cuda", generator=gen).float()       # kept as it is
    x[..., 0] = x[..., 32] = 127
    x *= 2.0 ** 100
    g = (torch.randn(4, 20, 1, 1, 64, dtype=torch.float64, device="cuda", generator=gen) * 2.0 ** power).float()
    got = checkpoint.weightGrad(g, checkpoint.compress(x))[..., 0, 0, 0].double()
    a, b = g.transpose(0, 1).reshape(20, -1).double(), x.transpose(0, 1).reshape(30, -1).double()
    limit = (8 + 16) * 2.0 ** -24 * (a.abs() @ b.abs().T) + 2.0 ** -133 * b.abs().sum(1)
    assert bool(((got - a @ b.T).abs() <= limit).all())


def test_weight_gradients_that_are_not_finite():
    """An infinity or NaN of the gradient is in all sums of its output, one of the input (kept as NaN) in those of its neuron, and in no others."""
    x, g = torch.ones(2, 30, 1, 1, 70, device="cuda"), torch.ones(2, 20, 1, 1, 70, device="cuda")
    g[0, 3, 0, 0, 69], g[1, 7, 0, 0, 0], x[1, 11, 0, 0, 40] = float("inf"), float("nan"), float("-inf")
    got = checkpoint.weightGrad(g, checkpoint.compress(x))[..., 0, 0, 0]
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[[3, 7]] = True
    bad[:, 11] = True
    assert torch.equal(got.isnan(), bad) and bool((got[~bad] == 140).all())
