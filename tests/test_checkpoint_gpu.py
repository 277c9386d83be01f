"""GPU: tensors kept in 8 bits, and the gradients formed from them, against their definitions in 64 bits.

What is kept is exact: equal to the definition, bit for bit.  The surrogate gradient: u - theta (half a step, 2^-24), the division
(half), exp (2 steps of 2^-23) and two products (half each): an argument z is off by 2^-23 |z|, so the result by (|z| + 4 + 2) 2^-23 of
itself, and 2^-126 where it is that small.  The weight gradient: a product of float32 and 8 bits in float32 precision is off
by 2^-24, and K of them are added up in parts of float32, whose roundings are random: less than 2^-24 (8 + sqrt(K)) of the sum of magnitudes."""
import math

import pytest
import torch

from slayerpytorch_b200 import checkpoint, layer

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NEURON = {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1}


def want_kept(x):
    """q 2^e from the definition, on the host"""
    rows, T = x.shape
    x = x.detach().cpu().double()
    out = torch.empty_like(x)
    for a in range(0, T, 32):
        part = x[:, a:a + 32]
        finite = part.isfinite()
        top = torch.where(finite, part.abs(), 0.0).amax(1)
        e = torch.tensor([max(-126, min(121, next((k for k in range(math.frexp(v)[1] - 9, math.frexp(v)[1] + 1) if v <= 127 * 2.0 ** k), 0))) if v else -126
                          for v in top.tolist()], dtype=torch.float64)[:, None]
        out[:, a:a + 32] = torch.where(finite, torch.clamp(torch.round(part / 2.0 ** e), -127, 127) * 2.0 ** e, float("nan"))
    return out


def same(got, value):
    """value, rounded to the type of got once"""
    assert torch.equal(got.isnan().cpu(), value.isnan())
    assert torch.equal(torch.where(got.isnan(), 0.0, got).cpu(), torch.where(value.isnan(), 0.0, value).to(got.dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,T", [(1, 1), (5, 3), (7, 31), (64, 32), (9, 33), (3, 64), (11, 100), (130, 145), (20, 300), (2, 4097)])
def test_what_is_kept(rows, T, dtype):
    gen = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, T, generator=gen) * torch.exp(3 * torch.randn(rows, 1, generator=gen))).to(dtype).cuda()
    kept = checkpoint.compress(x)
    assert kept.q.shape == (rows, (T + 31) // 32 * 32) and kept.shape == x.shape and kept.dtype == dtype
    assert bool((kept.q[:, T:] == 0).all())
    same(kept.restore(), want_kept(x))
    same(kept.restore(torch.float32), want_kept(x))
    same(kept.restore(torch.float16), want_kept(x))


def test_values_at_their_ends():
    inf, nan, most = float("inf"), float("nan"), 3.4028234663852886e38
    rows = [[0.0] * 32, [0.0, -0.0] * 16, [127.0] + [0.5, 1.5, 2.5, -0.5, -1.5] * 6 + [63.5], [127.0000001] * 32, [127.00001] + [1.0] * 31, [nan] * 32,
            [inf] + [1.0] * 31, [-inf, nan] + [1e-30] * 30, [most] * 32, [-most] + [1.0] * 31, [1e-45] * 32, [1e-38, 1e-40] * 16, [2.0 ** -126] * 32,
            [2.0 ** 121 * 127] * 32, [1e-37] * 31 + [1e30], [254.0, 1.0, 3.0, -1.0] * 8, [253.99998, 1.0, 3.0, -1.0] * 8]
    x = torch.tensor(rows, dtype=torch.float32).cuda()
    same(checkpoint.compress(x).restore(), want_kept(x))
    off = (checkpoint.compress(x).restore() - x).abs()
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(1, keepdim=True)
    assert bool((off <= torch.maximum(top / 127, torch.tensor(2.0 ** -127)))[x.isfinite()].all())


def test_shapes_strides_and_empty_tensors():
    x = torch.randn(2, 3, 4, 5, 50, device="cuda")
    kept = checkpoint.compress(x)
    assert kept.restore().shape == x.shape
    assert torch.equal(checkpoint.compress(x.transpose(0, 4).contiguous().transpose(0, 4)).q, kept.q)
    store = torch.zeros(x.numel() + 4, device="cuda")
    for off in (1, 2, 3):
        moved = store[off:off + x.numel()].view(x.shape)
        moved.copy_(x)
        assert torch.equal(checkpoint.compress(moved).q, kept.q)
    for shape in ((0, 5), (5, 0), (0,), (2, 0, 3)):
        empty = checkpoint.compress(torch.zeros(shape, device="cuda"))
        assert empty.restore().shape == shape
        assert checkpoint.spikeGrad(torch.zeros(shape, device="cuda"), empty, 1.0, 1.0, 1.0).shape == shape


@pytest.mark.parametrize("shape", [(1, 1), (7, 3, 1, 1, 31), (4, 512, 1, 1, 300), (3, 5, 6, 7, 301), (2, 3, 1450)])
@pytest.mark.parametrize("theta,tau,scale", [(10.0, 10.0, 1.0), (5120.0, 512.0, 0.3)])
def test_surrogate_gradient(shape, theta, tau, scale):
    gen = torch.Generator(device="cuda").manual_seed(1)
    u = theta * torch.randn(shape, device="cuda", generator=gen)
    g = torch.randn(shape, device="cuda", generator=gen)
    kept = checkpoint.compress(u)
    got = checkpoint.spikeGrad(g, kept, theta, tau, scale)
    z = (kept.restore().double() - theta).abs() / tau
    value = g.double() * scale / tau * torch.exp(-z)
    assert bool(((got.double() - value).abs() <= (z + 6) * 2.0 ** -23 * value.abs() + 2.0 ** -126).all())


def test_surrogate_gradient_of_what_is_not_finite():
    u = torch.zeros(2, 40, device="cuda")
    u[0, 5], u[1, 39] = float("nan"), float("inf")
    got = checkpoint.spikeGrad(torch.ones_like(u), checkpoint.compress(u), 1.0, 1.0, 1.0)
    assert bool(got[0, 5].isnan()) and bool(got[1, 39].isnan()) and int(got.isnan().sum()) == 2


def check_weight(N, O, sizes, T, seed, x=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if x is None:
        x = torch.randn(N, *sizes, T, device="cuda", generator=gen) * torch.exp(torch.randn(N, *sizes, 1, device="cuda", generator=gen))
    g = torch.randn(N, O, *(1,) * (len(sizes) - 1), T, device="cuda", generator=gen) * torch.exp(torch.randn(N, O, *(1,) * (len(sizes) - 1), T, device="cuda",
                                                                                                           generator=gen))
    kept = checkpoint.compress(x)
    got = checkpoint.weightGrad(g, kept)
    assert got.shape == (O, *sizes, 1) and got.dtype == torch.float32
    a = g.reshape(N, O, T).transpose(0, 1).reshape(O, -1).double()
    b = kept.restore(torch.float32).reshape(N, -1, T).transpose(0, 1).reshape(-1, N * T).double()
    value, size = a @ b.T, a.abs() @ b.abs().T
    wrong = (got.reshape(value.shape).double() - value).abs() - (8 + math.sqrt(N * T)) * 2.0 ** -24 * size
    assert bool((wrong <= 0).all()), float(wrong.max())
    assert torch.equal(got, checkpoint.weightGrad(g, kept))
    return g, kept, got


@pytest.mark.parametrize("N,O,sizes,T", [(1, 1, (1,), 1), (2, 3, (5,), 7), (3, 10, (4, 2, 3), 31), (1, 64, (64,), 32), (5, 65, (63,), 33), (2, 128, (256, 1, 1), 64),
                                         (4, 130, (300, 1, 1), 100), (8, 10, (512, 1, 1), 301), (64, 512, (37,), 20), (3, 513, (1030,), 145), (1, 200, (700,), 5000),
                                         (300, 33, (70,), 5), (2, 1024, (2, 20, 30), 96), (1, 1, (3000,), 70), (1, 700, (1,), 70), (17, 257, (129,), 64)])
def test_weight_gradient(N, O, sizes, T):
    check_weight(N, O, sizes, T, N + O)


@pytest.mark.parametrize("O,T", [(1, 1), (1, 2), (1, 3), (2, 1), (3, 1), (2, 3), (7, 1), (1, 7), (3, 5)])
@pytest.mark.parametrize("N", [1, 2, 3, 9, 20])
def test_weight_gradient_of_few_elements(N, O, T):
    """Samples of fewer elements than two loads of 16 bytes: the tensor ends within the reach of several."""
    check_weight(N, O, (5,), T, N + O + T)


def test_weight_gradient_at_its_ends():
    """Values of very different sizes, what is not finite, no samples, no steps."""
    x = torch.randn(3, 40, 70, device="cuda") * 2.0 ** torch.randint(-100, 30, (3, 40, 1), device="cuda")
    check_weight(3, 20, (40,), 70, 7, x)
    x[1, 7, 33] = float("nan")
    g, kept, got = check_weight_nan(x)
    assert bool(got[:, 7].isnan().all()) and int(got.isnan().sum()) == got.shape[0]
    g[0, 4, 69] = float("inf")
    got = checkpoint.weightGrad(g, kept)[..., 0]
    assert not bool(got[4].isfinite().any()) and int((~got.isfinite()).sum()) == 40 + 20 - 1
    for N, O, I, T in ((0, 3, 4, 5), (2, 3, 4, 0), (2, 0, 4, 5), (2, 3, 0, 5)):
        out = checkpoint.weightGrad(torch.zeros(N, O, T, device="cuda"), checkpoint.compress(torch.zeros(N, I, T, device="cuda")))
        assert out.shape == (O, I, 1) and bool((out == 0).all())


def check_weight_nan(x):
    g = torch.randn(3, 20, 70, device="cuda")
    kept = checkpoint.compress(x)
    return g, kept, checkpoint.weightGrad(g, kept)[..., 0]


def test_layers_that_keep_8_bits():
    """dense -> leak -> spike, forwards the same as without checkpoints, gradients as the formulas on what is kept say."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    net = layer.spikeLayer(NEURON, {"Ts": 1.0, "tSample": 90}).cuda()
    dense, plain = net.dense((6, 5, 2), 11, checkpoint=True).cuda(), net.dense((6, 5, 2), 11).cuda()
    plain.load_state_dict(dense.state_dict())
    x = torch.rand(3, 2, 5, 6, 90, device="cuda", generator=gen)
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    y, z = dense(leaf), plain(other)
    assert torch.equal(y, z)
    g = torch.randn(y.shape, device="cuda", generator=gen)
    y.backward(g), z.backward(g)
    assert torch.allclose(leaf.grad, other.grad, rtol=1e-5, atol=1e-4)
    assert torch.equal(dense.weight.grad, checkpoint.weightGrad(g, checkpoint.compress(x)))
    # 8 bits: off by 1/254 to 1/127 of each group's largest value (1 at most here)
    size = (g.reshape(3, 11, 90).abs().sum((0, 2)) / 127)[:, None, None, None, None]
    assert bool(((dense.weight.grad - plain.weight.grad).abs() <= size * 1.1).all())
    with pytest.raises(ValueError, match="inputs of its own size"):
        dense(torch.zeros(1, 2, 6, 6, 9, device="cuda"))

    u = 8.0 * torch.randn(3, 11, 1, 1, 90, device="cuda", generator=gen)
    a, b = u.clone().requires_grad_(), u.clone().requires_grad_()
    s, t = net.spike(a.clone(), checkpoint=True), net.spike(b.clone())
    assert torch.equal(s, t)
    h = torch.randn(s.shape, device="cuda", generator=gen)
    (ga,), (gb,) = torch.autograd.grad(s, [a], h), torch.autograd.grad(t, [b], h)
    after = u.clone()
    layer.slayerCuda.getSpikes(after, net.refKernel, 10.0, 1.0)
    assert torch.equal(ga, checkpoint.spikeGrad(h, checkpoint.compress(after), 10.0, 10.0, 1.0))
    # an error of top / 127 in u changes log rho by that over tau
    top = torch.nn.functional.max_pool1d(after.reshape(33, 1, 90).abs(), 32, 32, ceil_mode=True).repeat_interleave(32, -1)[..., :90].reshape(u.shape)
    assert bool(((ga - gb).abs() <= gb.abs() * (torch.exp(top / 127 / 10) - 1) * 1.01 + 1e-9).all())
    # what needs no gradient keeps nothing and runs
    with torch.no_grad():
        assert torch.equal(net.spike(u.clone(), checkpoint=True), s)


def test_a_network_of_them():
    """A step of training over a longer sequence, captured and replayed, gives the eager step's gradients."""
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
    assert all(bool(v.isfinite().all()) for v in eager) and all(float(v.abs().max()) > 0 for v in eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for v in out:
        v.detach().zero_()
    graph.replay()
    assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]) and torch.equal(out[3], eager[3])


def test_refusals():
    x = torch.zeros(2, 3, 40, device="cuda")
    kept = checkpoint.compress(x)
    for call in (lambda: checkpoint.spikeGrad(x[..., :39], kept, 1.0, 1.0, 1.0), lambda: checkpoint.weightGrad(x[:1], kept),
                 lambda: checkpoint.weightGrad(x[..., None, :].expand(2, 3, 2, 40), kept), lambda: checkpoint.compress(x[0, 0, 0]),
                 lambda: checkpoint.weightGrad(x[0], checkpoint.compress(x[0])),
                 lambda: checkpoint.Checkpoint(kept.q[:1], kept.scale, kept.shape, kept.dtype).restore(),
                 lambda: checkpoint.Checkpoint(kept.q, kept.scale[:, :1], kept.shape, kept.dtype).restore()):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: checkpoint.compress(x.double()), lambda: checkpoint.compress(x.cpu()), lambda: checkpoint.spikeGrad(x.half(), kept, 1.0, 1.0, 1.0),
                 lambda: checkpoint.weightGrad(x.half(), kept), lambda: kept.restore(torch.int32),
                 lambda: checkpoint.Checkpoint(kept.q.cpu(), kept.scale.cpu(), kept.shape, kept.dtype).restore(),
                 lambda: checkpoint.Checkpoint(kept.q.int(), kept.scale, kept.shape, kept.dtype).restore()):
        with pytest.raises(RuntimeError):
            call()
