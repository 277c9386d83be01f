"""GPU: the gradient of gates that rows share, added up over few and over many rows, of few and of many gates."""
import pytest
import torch

from slayerpytorch_b200.recurrence import gatedLeak
from test_leak_gpu import STEP, check, made

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,C,T,shape", [
    (1, 1000, 8, (1000, 1)), (2, 777, 5, (777, 1)), (16, 100, 7, (100, 1)), (17, 100, 7, (100, 1)), (512, 33, 4, (33, 1)), (513, 33, 4, (33, 1)),
    (40, 3, 2, (40, 3, 1)), (9, 15, 16, (9, 1, 1)), (9, 16, 16, (9, 1, 1)), (300, 31, 6, (300, 1, 1)), (300, 32, 6, (300, 1, 1)), (5, 511, 9, (5, 1, 1)),
    (5, 513, 9, (5, 1, 1)), (1, 9000, 3, (1, 1)), (1, 1, 300, (1, 1)), (1, 1, 20000, (1, 1)), (3, 5, 20000, (5, 1)), (2, 40, 9000, (40, 1)), (3, 4, 9000, (3, 1, 1)),
    (4, 3000, 1, (3000, 1)),
    (40, 1300, 3, (1300, 1)), (17, 2001, 2, (2001, 1)), (1300, 17, 3, (1300, 1, 1)), (1300, 40, 2, (1300, 1, 1))])
def test_sums_over_rows(N, C, T, shape):
    """From one number a gate to more than a CTA has; gates of rows that lie together, that do not, and of rows that are split."""
    x, gate, h, g, gs, gen = made(N, C, T, torch.float32, 'logit', N + C, shape)
    check(x, gate, h, None, 'logit', True, g, gs)
    check(x, gate, h, torch.randint(0, T + 1, (N,), device="cuda", generator=gen), 'logit', False, g, gs)


def test_gates_of_images():
    """One for each channel or pixel of images: rows of a gate lie together (inner dimensions) and apart (samples)."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g = (torch.randn(6, 7, 5, 3, 12, device="cuda", generator=gen) for _ in range(2))
    for shape in ((7, 1, 1, 1), (7, 5, 1, 1), (7, 5, 3, 1), (6, 7, 1, 1, 1), (1, 1, 1, 1), (5, 3, 1), (3, 1)):
        gate = torch.randn(shape, device="cuda", generator=gen).requires_grad_()
        (got,) = torch.autograd.grad(gatedLeak(x, gate), [gate], g)
        full = gate.detach().expand_as(x).contiguous().requires_grad_()
        (each,) = torch.autograd.grad(gatedLeak(x, full), [full], g)
        want, size = (v.double().sum_to_size((1,) * (5 - len(shape)) + shape).reshape(shape) for v in (each, each.abs()))
        # the same terms, whose decays and states are rounded otherwise: both off by as much as a lane's 12 steps and its maps are (test_leak_gpu.py)
        assert bool(((got.double() - want).abs() <= 2 * 200 * STEP * size).all())


def test_millions_of_gates():
    """Every gate gets its own sum, and the same in every call."""
    C, T = 3000001, 3
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, g = (torch.randn(1, C, T, device="cuda", generator=gen) for _ in range(2))
    gate = torch.randn(C, 1, device="cuda", generator=gen).requires_grad_()
    (a,) = torch.autograd.grad(gatedLeak(x, gate), [gate], g)
    (b,) = torch.autograd.grad(gatedLeak(x, gate), [gate], g)
    assert torch.equal(a, b)
    f, x, g = torch.sigmoid(gate.detach().double())[:, 0], x[0].double(), g[0].double()
    y0, l2 = x[:, 0], g[:, 2]
    y1, l1 = f * y0 + x[:, 1], f * l2 + g[:, 1]
    want = (l1 * y0 + l2 * y1) * f * (1 - f)
    size = ((f * l2.abs() + g[:, 1].abs()) * y0.abs() + l2.abs() * (f * y0.abs() + x[:, 1].abs())) * f * (1 - f)
    # decays are off by (8 + |gate|) steps each, slopes, states and products by a few
    assert bool(((a[:, 0].double() - want).abs() <= (4 * (8 + gate.detach()[:, 0].abs()) + 20) * STEP * size + 1e-37).all())


@pytest.mark.parametrize("rows,T", [(2000000, 4), (3, 20000)])
def test_a_forward_pass_needs_no_memory_for_the_gates_gradients(rows, T):
    """Beside its result: nothing, or, of rows that are split, 16 bytes for each segment and row at most."""
    x, gate = torch.randn(1, rows, T, device="cuda"), torch.randn(rows, 1, device="cuda")
    with torch.no_grad():
        gatedLeak(x, gate)
        torch.cuda.reset_peak_memory_stats()
        asked = lambda which: torch.cuda.memory_stats()["requested_bytes.all." + which]  # noqa: E731
        before = asked("current")
        y = gatedLeak(x, gate)
        assert asked("peak") - before <= y.numel() * 4 + (rows * 40 * 16 + 64 if T > 512 else 0)
