"""GPU: the losses of choices at their edges - logits filled with large values, margins without bound, empty inputs, many rows.

Tolerances.  A row's sum of exponentials 2^((x - m) k) is held in fp32.  The argument d has up to three roundings of 2^-24 |d| (the
difference, the product, k itself), which weigh on the sum as 3 ln 2 2^-24 E|d|, with E|d| <= log2(V) + 1 < 17: 2.2e-6; the exponential's
own error is 2^-22; a running sum is raised to a new maximum at most 32 times (a lane of a short row; long rows 10 times) at
2^-22 + 2^-24 each, 9.6e-6, and added to as often, 2e-6.  Together 1.4e-5 < SUM = 1.5e-5.  A softmax entry of more than
2^-126 has its own exponential's 3 ln 2 2^-24 126 = 1.6e-5 on top of that: with the roundings of the coefficient and the product
below REL = 4e-5 of |c| (delta + p).  The result's rounding is half a step of its type (`close`)."""
import math

import pytest
import torch

from slayerpytorch_b200 import loss
from tests.test_choices_gpu import CLIP, SUM, TYPES, close, descriptor, policy_want, want_grad, want_logp

pytestmark = pytest.mark.gpu

FILLS = [-1e4, -1e9, -1e10, -1e12, -1e20, -1e30, -1e36, -3.3895e38]


def of_ratio(x, action, size, scale):
    """What a gradient is off by where a coefficient made of `size` has its ratio from a log-probability that is off by SUM."""
    p = torch.softmax(x.double() * scale, -1)
    return scale * (size * SUM)[..., None] * (torch.zeros_like(p).scatter_(-1, action[..., None], 1.0) + p)


def filled(V, dtype, seed):
    """Rows of ordinary logits in which something is filled: (logits, an entry that is not)"""
    gen = torch.Generator().manual_seed(seed)
    fills = [f for f in FILLS if f >= torch.finfo(dtype).min] + [torch.finfo(dtype).min]
    rows, action = [], []
    for f in fills:
        for where in (slice(0, 1), slice(V - 1, V), slice(0, V // 2), slice(V // 2, V), slice(1, V, 2), slice(0, V - 1)):
            x = torch.randn(V, generator=gen) * 3
            x[where] = f
            left = (x > -1e3).nonzero()[:, 0]
            rows.append(x)
            action.append(left[torch.randint(0, len(left), (1,), generator=gen)])
    x = torch.stack(rows).to(dtype)
    return x, torch.cat(action), gen


@pytest.mark.parametrize("scale", [1.0, 0.7, 0.2])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [10, 300, 5003, 40003])
def test_filled_entries(V, dtype, scale):
    """Illegal actions, a padded vocabulary, all but one entry: any finite fill leaves the row what it is without these entries."""
    x, action, gen = filled(V, dtype, V)
    up = torch.randn(len(x), generator=gen)
    for rows in (slice(0, len(x)), slice(0, 12)):            # a CTA for each row; a cluster for each
        leaf = x[rows].cuda().requires_grad_()
        lp = loss.actionLogProb(leaf, action[rows].cuda(), scale=scale)
        (g,) = torch.autograd.grad(lp, [leaf], up[rows].cuda())
        close(lp.detach(), want_logp(x[rows], action[rows], scale), SUM)
        close(g, *want_grad(x[rows], action[rows], up[rows].double(), scale))
    lp = want_logp(x, action, scale)
    old = (lp - torch.randint(0, 2, (len(x),), generator=gen) * 0.1 + 0.05).float()
    adv = torch.randn(len(x), generator=gen)
    leaf = x.cuda().requires_grad_()
    got = loss.policyLoss(leaf, action.cuda(), old.cuda(), adv.cuda(), clip=CLIP, scale=scale)
    (g,) = torch.autograd.grad(got, [leaf])
    value, slack, coef, size = policy_want(x[:, None], action[:, None], old[:, None], adv[:, None], None, None, 0.0, "sum", scale)
    assert abs(float(got.detach()) - float(value)) <= float(slack) + 2 ** -24 * abs(float(value))
    grad, spare = want_grad(x, action, coef[:, 0], scale)
    close(g, grad, spare + of_ratio(x, action, size[:, 0], scale))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [10, 300, 5003, 40003])
def test_rows_of_equal_entries_of_any_size(V, dtype):
    values = [s * 10.0 ** e for e in (0, 3, 4, 5, 6, 8, 9, 10, 12, 20, 30, 36, 37, 38) for s in (1, -1)]
    x = torch.tensor(values)[:, None].expand(-1, V).to(dtype)
    action = torch.arange(len(values)) % V
    for scale in (1.0, 0.3, 7.0):
        leaf = x.cuda().requires_grad_()
        lp = loss.actionLogProb(leaf, action.cuda(), scale=scale)
        (g,) = torch.autograd.grad(lp.sum(), [leaf])
        close(lp.detach(), torch.full((len(values),), -math.log(V), dtype=torch.float64), SUM)
        close(g, *want_grad(x, action, torch.ones(len(values), dtype=torch.float64), scale))


@pytest.mark.parametrize("V", [10, 300, 5003, 40003])
@pytest.mark.parametrize("top", [1e3, 1e4, 1.2e4, 1e5, 1e6, 1e7, 1e8, 1e12])
def test_policy_value_and_gradient_have_one_ratio(top, V):
    """Rows that lie far from zero: the gradient's ratio is the loss's, as near to 64 bits as anywhere."""
    gen = torch.Generator().manual_seed(int(top))
    step = max(1.0, top * 2.0 ** -23)                         # the entries are a few steps of float32 apart
    scale = 0.9 / step
    x = top + 3 * step * torch.randn(24, 1, V, generator=gen, dtype=torch.float64)
    x = torch.cat([x, -x]).float()
    action = torch.randint(0, V, (48, 1), generator=gen)
    lp = want_logp(x, action, scale)
    ratio = torch.tensor([0.3, 0.7, 0.95, 1.0, 1.1, 1.22, 2.5], dtype=torch.float64)[torch.randint(0, 7, (48, 1), generator=gen)]
    old = (lp - ratio.log()).float()
    ref = (lp + 0.5 * torch.randn(48, 1, generator=gen)).float()
    adv = torch.randn(48, 1, generator=gen)
    leaf = x.cuda().requires_grad_()
    got = loss.policyLoss(leaf, action.cuda(), old.cuda(), adv.cuda(), refLogProb=ref.cuda(), clip=CLIP, klCoef=0.3, scale=scale)
    (g,) = torch.autograd.grad(got, [leaf])
    scale = float(torch.tensor(scale, dtype=torch.float32))   # what the kernels take it as
    value, slack, coef, size = policy_want(x, action, old, adv, ref, None, 0.3, "sum", scale)
    # |gap| <= 30 here: the scale's rounding is in `scale` itself
    assert abs(float(got.detach()) - float(value)) <= float(slack) + 2 ** -24 * abs(float(value))
    grad, spare = want_grad(x, action, coef, scale)
    close(g, grad, spare + of_ratio(x, action, size, scale))


def test_preference_of_impossible_choices():
    """A choice of probability zero in one sequence of a pair: h is without bound, the slopes are its limits, and a term of weight 0 is 0."""
    inf = float("inf")
    for V in (6, 2000):
        gen = torch.Generator().manual_seed(V)
        x = torch.randn(4, 3, V, generator=gen)
        action = torch.randint(1, V, (4, 3), generator=gen)
        ref = torch.randn(4, generator=gen)
        lp = want_logp(x, action).sum(1) - ref.double()
        for at, smoothing in ((0, 0.0), (2, 0.0), (0, 0.25), (2, 0.25), (0, 1.0), (2, 1.0)):        # the preferred one's, the rejected one's
            y = x.clone()
            y[at, 1, action[at, 1]] = -inf
            leaf = y.cuda().requires_grad_()
            got = loss.preferenceLoss(leaf, action.cuda(), ref.cuda(), beta=0.4, labelSmoothing=smoothing)
            (g,) = torch.autograd.grad(got, [leaf])
            h = 0.4 * float(lp[1] - lp[3])
            other = (1 - smoothing) * math.log1p(math.exp(-h)) + smoothing * math.log1p(math.exp(h))
            weight = 1 - smoothing if at == 0 else smoothing        # of the side that has no bound
            if weight:
                assert float(got.detach()) == inf
            else:
                assert abs(float(got.detach()) - other) <= 0.8 * 3 * (SUM + 2 ** -24 * 20) + 2 ** -23 * other
            slope = 0.4 * ((0.0 if at == 0 else 1.0) - (1 - smoothing))
            rest = 0.4 * (1 / (1 + math.exp(-h)) - (1 - smoothing))
            coef = torch.tensor([slope, rest, -slope, -rest], dtype=torch.float64)[:, None].expand(4, 3)
            grad, spare = want_grad(y, action, coef)
            p = torch.softmax(y.double(), -1)
            delta = torch.zeros_like(p).scatter_(-1, action[..., None], 1.0)
            # a slope is off by beta^2 / 4 of what the margins are off by
            close(g, grad, spare + 0.04 * 2 * 3 * (SUM + 2 ** -24 * 20) * (delta + p))


@pytest.mark.parametrize("V", [10, 300, 5003, 40003])
def test_choices_far_below_the_maximum(V):
    """The distance of the chosen entry from the maximum is not rounded on the way (it may not even be a float32)."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(64, V, generator=gen)
    action = torch.randint(1, V, (64,), generator=gen)
    x[:, 0] = 3000.0 + 40.0 * torch.rand(64, generator=gen)
    x[0, 0], x[0, action[0]] = 3e38, -3e38
    x[1, 0], x[1, action[1]] = 1e30, -2e38
    # the maximum is all there is to the sum: off by its own exponential's 2^-22 and the sum's rounding; then one rounding of the result
    for scale in (0.1, 0.4):
        lp = loss.actionLogProb(x.cuda(), action.cuda(), scale=scale)
        exact = float(torch.tensor(scale, dtype=torch.float32))
        close(lp, want_logp(x, action, exact), 2.0 ** -21)


@pytest.mark.parametrize("V", [9, 1500])
def test_the_returned_log_probabilities_are_the_callers_own(V):
    gen = torch.Generator().manual_seed(V)
    x, action = torch.randn(3, 4, V, generator=gen), torch.randint(0, V, (3, 4), generator=gen)
    z = torch.zeros(3, 4, device="cuda")
    leaf = x.cuda().requires_grad_()
    want = torch.autograd.grad(loss.policyLoss(leaf, action.cuda(), z - 2, z + 1), [leaf])[0]
    value, lp = loss.policyLoss(leaf, action.cuda(), z - 2, z + 1, returnLogProb=True)
    kept = lp.clone()
    lp.add_(5.0).exp_()                                       # written over before the backward passes
    for up in (1.0, 1.0, 2.0):
        (g,) = torch.autograd.grad(value * up, [leaf], retain_graph=True)
        assert torch.equal(g, want * up)
    close(kept, want_logp(x, action), SUM)
    # and it holds no more than its rows
    assert lp.untyped_storage().nbytes() <= 4 * 12 + 512


@pytest.mark.parametrize("reduction", ["sum", "mean", "sequence"])
def test_sequences_without_choices_and_one_advantage_each(reduction):
    leaf = torch.zeros(4, 0, 7, device="cuda", requires_grad=True)
    none = torch.zeros(4, 0, device="cuda")
    got = loss.policyLoss(leaf, none.long(), none, torch.ones(4, device="cuda"), reduction=reduction)
    (g,) = torch.autograd.grad(got, [leaf])
    assert float(got.detach()) == 0.0 and g.shape == leaf.shape


def test_spike_losses_of_no_samples():
    d = descriptor("Policy")
    spikes = torch.zeros(0, 7, 1, 1, 50, device="cuda", requires_grad=True)
    none = torch.zeros(0, device="cuda")
    net = loss.spikeLoss(d).cuda()
    assert net.actionLogProb(spikes, none.long()).shape == (0,)
    got = net.policy(spikes, none.long(), none, none)
    (g,) = torch.autograd.grad(got, [spikes])
    assert float(got.detach()) == 0.0 and g.shape == spikes.shape
    net = loss.spikeLoss(descriptor("Preference")).cuda()
    for shape, value in (((0, 3), 0.0), ((2, 0), math.log(2.0))):
        got = net.preference(spikes, none.long().reshape(shape), torch.zeros(shape[0], device="cuda"))
        (g,) = torch.autograd.grad(got, [spikes])
        assert abs(float(got.detach()) - value) < 1e-6 and g.shape == spikes.shape


def check_policy(x, action, old, ref, adv, mask, up, scale=0.9):
    """A multiple of the policy loss, its log-probabilities and its gradient (all on the device)"""
    leaf = x.detach().requires_grad_()
    got, lp = loss.policyLoss(leaf, action, old, adv, refLogProb=ref, mask=mask, clip=CLIP, klCoef=0.3, scale=scale, returnLogProb=True)
    (g,) = torch.autograd.grad(got * up, [leaf])
    value, slack, coef, size = policy_want(x, action, old, adv, ref, mask, 0.3, "sum", scale)
    assert abs(float(got.detach()) - float(value)) <= float(slack) + 2 ** -24 * abs(float(value))
    close(lp, torch.where(mask, want_logp(x, action, scale), 0.0).cpu(), SUM)
    assert bool((g[~mask] == 0).all())
    for r in range(0, len(x), 400):
        part = slice(r, r + 400)
        grad, spare = want_grad(x[part], action[part], up * coef[part], scale)
        close(g[part], grad.cpu(), (spare + abs(up) * of_ratio(x[part], action[part], size[part], scale)).cpu())


def many_rows(rows, V, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, 1, V, generator=gen, device="cuda") * 3).to(dtype)
    action = torch.randint(0, V, (rows, 1), generator=gen, device="cuda")
    lp = torch.cat([want_logp(x[r:r + 400], action[r:r + 400], 0.9) for r in range(0, rows, 400)])
    ratio = torch.tensor([0.3, 0.7, 0.95, 1.0, 1.1, 1.22, 2.5], dtype=torch.float64, device="cuda")[torch.randint(0, 7, (rows, 1), generator=gen, device="cuda")]
    old = (lp - ratio.log()).float()
    ref = (lp + 0.5 * torch.randn(rows, 1, generator=gen, device="cuda")).float()
    adv = torch.randn(rows, 1, generator=gen, device="cuda")
    mask = torch.rand(rows, 1, generator=gen, device="cuda") < 0.6
    mask[1183:1187] = torch.tensor([[True], [False], [False], [True]], device="cuda")
    return x, action, old, ref, adv, mask


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1030, 4097])
@pytest.mark.parametrize("up", [1.0, 0.5])
def test_policy_more_long_rows_than_a_rescaled_gradient_has_ctas(up, V, dtype):
    """The gradient of a loss that was multiplied by something is formed by at most eight CTAs per SM, which walk over the rows."""
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count * 2 + 77
    check_policy(*many_rows(rows, V, dtype, V), up)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,per_cta", [(7, 32), (32, 32), (33, 8), (80, 8)])
@pytest.mark.parametrize("up", [1.0, 0.5])
def test_policy_more_short_rows_than_ctas_hold(up, V, per_cta, dtype):
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count * per_cta + 1001
    check_policy(*many_rows(rows, V, dtype, V), up)


def test_more_than_2_to_31_logits():
    rows, V = 70001, 32768
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(rows, V, generator=gen, device="cuda", dtype=torch.bfloat16)
    action = torch.randint(0, V, (rows,), generator=gen, device="cuda")
    leaf = x.requires_grad_()
    lp = loss.actionLogProb(leaf, action)
    up = torch.randn(rows, generator=gen, device="cuda")
    (g,) = torch.autograd.grad(lp, [leaf], up)
    for part in (slice(0, 3), slice(65530, 65545), slice(rows - 3, rows)):
        y = x.detach()[part]
        close(lp.detach()[part], want_logp(y, action[part]).cpu(), SUM)
        grad, spare = want_grad(y, action[part], up[part].double())
        close(g[part], grad.cpu(), spare.cpu())
