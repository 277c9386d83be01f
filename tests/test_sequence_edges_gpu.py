"""GPU: the gated leak and tensors in 8 bits at their edges - offsets past 32 bits, streams and graphs side by side, the order of rows, exact powers."""
import pytest
import torch

from slayerpytorch_b200 import capi, checkpoint, layer
from slayerpytorch_b200.recurrence import gatedLeak, gatedLeakStep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [8, 300, 2000])
def test_leaks_of_more_than_2_to_31_elements(T):
    """A row's result does not depend on where it lies: the last rows equal those of a call of their own."""
    rows = (1 << 31) // T + 4096
    x = torch.empty(rows, T, dtype=torch.bfloat16, device="cuda").normal_()
    gate = torch.full((1,), 2.0, device="cuda").expand(rows).reshape(rows, 1).contiguous()
    last = x[-4096:].clone()
    y = gatedLeak(x, gate, coupled=True)
    assert torch.equal(y[-4096:], gatedLeak(last, gate[-4096:], coupled=True))
    del y
    leaf, own = x.requires_grad_(), last.requires_grad_()
    (a,) = torch.autograd.grad(gatedLeak(leaf, gate), [leaf], x.detach())
    (b,) = torch.autograd.grad(gatedLeak(own, gate[-4096:]), [own], last.detach())
    assert torch.equal(a[-4096:], b)


def test_tensors_in_8_bits_of_more_than_2_to_31_elements():
    for T in (300, 301):
        rows = (1 << 31) // T + 4096
        x = torch.empty(rows, T, dtype=torch.bfloat16, device="cuda").normal_()
        kept = checkpoint.compress(x)
        own = checkpoint.compress(x[-4096:].clone())
        assert torch.equal(kept.q[-4096:], own.q) and torch.equal(kept.scale[:, -4096:], own.scale)
        assert torch.equal(kept.restore()[-4096:], own.restore())
        u = torch.empty(rows, T, device="cuda").normal_()
        got = checkpoint.spikeGrad(u, kept, 1.0, 1.0, 1.0)
        assert torch.equal(got[-4096:], checkpoint.spikeGrad(u[-4096:].clone(), own, 1.0, 1.0, 1.0))
        del x, kept, u, got


@pytest.mark.parametrize("N,O,I,T", [(70000, 2, 1000, 32), (40000, 1800, 3, 31)])
def test_weight_gradients_of_more_than_2_to_31_elements(N, O, I, T):
    """Only the last samples' gradients are not zero: the result is theirs, up to the order of sums."""
    x = torch.randint(-100, 101, (N, I, T), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    g = torch.zeros(N, O, T, device="cuda")
    g[-3:].normal_()
    kept = checkpoint.compress(x)
    got = checkpoint.weightGrad(g, kept)
    a = g[-3:].transpose(0, 1).reshape(O, -1).double()
    b = checkpoint.compress(x[-3:].clone()).restore(torch.float32).transpose(0, 1).reshape(I, -1).double()
    # three times T products of float32 precision
    assert bool(((got[..., 0].double() - a @ b.T).abs() <= (8 + (3 * T) ** 0.5) * 2.0 ** -24 * (a.abs() @ b.abs().T)).all())


def test_streams_side_by_side():
    """Calls of all operators on four streams at once give what they give one after the other."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    data = [(torch.randn(3, 40, 1, 1, 5000, device="cuda", generator=gen), torch.randn(3, 40, 1, 1, 5000, device="cuda", generator=gen),
             torch.randn(3, 300, 1, 1, 5000, device="cuda", generator=gen)) for _ in range(4)]

    def work(x, gate, g):
        y, s = gatedLeak(x, gate, returnState=True)
        kept = checkpoint.compress(y)
        return [y, s, kept.restore(), checkpoint.spikeGrad(x, kept, 1.0, 2.0, 1.0), checkpoint.weightGrad(g, kept)]
    alone = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    out = []
    for s, d in zip(streams, data):
        with torch.cuda.stream(s):
            out.append([work(*d) for _ in range(3)])
    torch.cuda.synchronize()
    for a, runs in zip(alone, out):
        for b in runs:
            assert all(torch.equal(v, w) for v, w in zip(a, b))
    assert capi.device_status() == 0


def test_two_graphs():
    """Two captured graphs, replayed in turn and on two streams, each with workspaces of its own."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    made = []
    for k in range(2):
        x, gate = (torch.randn(1, 3, 20000, device="cuda", generator=gen) for _ in range(2))
        g = torch.randn(1, 70, 20000, device="cuda", generator=gen)
        eager = [gatedLeak(x, gate), checkpoint.weightGrad(g, checkpoint.compress(x))]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [gatedLeak(x, gate), checkpoint.weightGrad(g, checkpoint.compress(x))]
        made.append((graph, eager, out, x, gate, g))
    side = torch.cuda.Stream()
    for _ in range(3):
        made[0][0].replay()
        with torch.cuda.stream(side):
            made[1][0].replay()
    torch.cuda.synchronize()
    for graph, eager, out, *_ in made:
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_rows_do_not_depend_on_one_another():
    """The same rows in another order, and rows of T steps as the start of longer ones."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for T in (7, 100, 301, 1500):
        x, gate = (torch.randn(64, T, device="cuda", generator=gen) for _ in range(2))
        order = torch.randperm(64, device="cuda", generator=gen)
        y, z = gatedLeak(x, gate), gatedLeak(x[order], gate[order])
        assert torch.allclose(y[order], z, rtol=0, atol=float(y.abs().max()) * 2.0 ** -20)
        if T % 4 == 0:          # lanes begin at the same steps
            assert torch.equal(y[order], z)
        kept, other = checkpoint.compress(x), checkpoint.compress(x[order])
        assert torch.equal(kept.q[order], other.q) and torch.equal(kept.scale[:, order], other.scale)


@pytest.mark.parametrize("kind", ['logit', 'decay'])
def test_a_stop_forgets_everything(kind):
    """A step that keeps nothing stops whatever was before it, however large, for the rest of the row, wherever it lies."""
    stop = float("-inf") if kind == 'logit' else 0.0
    for T in (40, 300, 513, 3000):
        for at in {0, 1, 15, 16, 17, 31, 39, T // 2, T - 1}:
            x, gate = torch.ones(2, T, device="cuda"), torch.full((2, T), 5.0 if kind == 'logit' else 0.99, device="cuda")
            x[1, :at], gate[:, at] = 1e30, stop
            # (a call for each: in one, rows of odd lengths lie differently, and lanes begin at other steps)
            y, z = (gatedLeak(x[i:i + 1].clone(), gate[i:i + 1].clone(), kind=kind, initial=torch.tensor([h], device="cuda"))
                    for i, h in ((0, 0.0), (1, 1e35)))
            assert torch.equal(y[0, at:], z[0, at:]) and float(z[0, at]) == 1.0


def test_single_steps_of_a_long_stream():
    """Ten thousand steps with a slow leak: states are rounded to 32 bits each time, half a step at random."""
    gate = torch.tensor([8.0, 5.0, -2.0, 12.0], device="cuda")
    f = torch.sigmoid(gate.double())
    state, want = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda")
    x = torch.ones(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gatedLeakStep(x, gate, state)
    for _ in range(10000):
        graph.replay()
        want = f * want + 1
    # one minus f is known to (8 + |gate|) 2^-24; roundings of up to 10000 states, 2^-24 each, at random: less than 500 of them
    assert bool(((state.double() - want).abs() <= (8 + gate.abs() + 500) * 2.0 ** -24 * want).all())


def test_a_gate_of_another_type_on_one_step():
    """A sequence of one step, of one sample: a float32 gate per neuron has as many elements as x then, and is taken as for longer ones."""
    gate, h = torch.linspace(-3, 3, 5, device="cuda"), torch.linspace(1, 2, 5, device="cuda").reshape(1, 5)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.linspace(-1, 1, 10, device="cuda").reshape(2, 5, 1).to(dtype)
        leaf = gate.clone().requires_grad_()
        y = gatedLeak(x, leaf[None, :, None], initial=h.expand(2, 5))
        (whole,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        for i in range(2):
            one = gatedLeak(x[i:i + 1], leaf[None, :, None], initial=h)
            # a float32 gate of one step is taken as one for each step, whose decay is formed otherwise: two decays, each off by (8 + |gate|)
            # 2^-24 of itself, of a state of up to 2, and two roundings of results of up to 3 each
            assert torch.allclose(one, y[i:i + 1], rtol=0, atol=(2 * (8 + 3) * 2 + 4 * 3) * 2.0 ** -24 if dtype == torch.float32 else 0)
            (part,) = torch.autograd.grad(one, leaf, torch.ones_like(one))
            # one sample's share, h f (1 - f): x has no part in it; f and 1 - f as above, on both sides, and eight roundings
            assert part.dtype == torch.float32 and torch.allclose(2 * part, whole, rtol=(4 * (8 + 3) + 8) * 2.0 ** -24, atol=0)
            state = h.clone()
            step = gatedLeakStep(x[i:i + 1, :, 0], gate[None], state)
            assert torch.allclose(step.float(), one[..., 0].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)


def test_a_state_apart_from_what_is_read():
    """One buffer may hold state, x and gate, but not in the same places."""
    buffer = torch.rand(40, device="cuda")
    x, gate, state = buffer[:10], buffer[10:20], buffer[20:30]
    want = torch.sigmoid(gate.double()) * state.double() + x.double()
    assert torch.allclose(gatedLeakStep(x, gate, state).double(), want, rtol=16 * 2.0 ** -24, atol=0)
    for bad in ((buffer[15:25], gate), (x, buffer[29:39]), (x, state[:1]), (state, gate)):
        before = buffer.clone()
        with pytest.raises(ValueError, match="share memory"):
            gatedLeakStep(*bad, state)
        assert torch.equal(buffer, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("auto", [False, True])
def test_dense_layers_in_16_bits(dtype, auto):
    """A layer of 16-bit weights, or one under autocast, keeps its input in 8 bits too; its gradients are those of what is kept, in 32 bits."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    net = layer.spikeLayer({"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1},
                           {"Ts": 1.0, "tSample": 50})
    dense, plain = net.dense(30, 12, checkpoint=True).cuda(), net.dense(30, 12).cuda()
    plain.load_state_dict(dense.state_dict())
    kind = torch.float32 if auto else dtype
    dense, plain = dense.to(kind), plain.to(kind)
    x = torch.randint(-127, 128, (3, 30, 1, 1, 50), device="cuda", generator=gen).to(kind)      # kept as it is
    x[..., 0] = 127
    x[..., 32] = 127
    leaf = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=dtype, enabled=auto):
        y, z = dense(leaf), plain(x)
    assert y.dtype == z.dtype == dtype and torch.equal(y, z)
    g = torch.randn(y.shape, device="cuda", generator=gen).to(dtype)
    y.backward(g)
    assert leaf.grad.dtype == dense.weight.grad.dtype == kind
    # weights: 150 products each, in 32 bits
    a, b = g.transpose(0, 1).reshape(12, -1).double(), x.transpose(0, 1).reshape(30, -1).double()
    half = torch.finfo(kind).eps / 2
    want = (a @ b.T).reshape(dense.weight.shape)
    assert bool(((dense.weight.grad.double() - want).abs() <= half * 1.01 * want.abs() + (8 + 150 ** 0.5) * 2.0 ** -24 * (a.abs() @ b.abs().T).reshape(want.shape)).all())
    # inputs: 12 products each, rounded to 16 bits (float16: also to whole multiples of 2^-24)
    w, up = dense.weight.to(dtype).double().reshape(12, 30), g.double().reshape(3, 12, 50)
    back, size = torch.einsum("oi,not->nit", w, up), torch.einsum("oi,not->nit", w.abs(), up.abs())
    half = torch.finfo(dtype).eps / 2
    assert bool(((leaf.grad.double().reshape(back.shape) - back).abs() <= half * 1.01 * back.abs() + 13 * 2.0 ** -24 * size + 2.0 ** -25).all())
