"""GPU: the losses of choices (rows of logits, one entry each) against their definitions in 64 bits.

Tolerances.  The kernels hold a row's sum of exponentials in fp32: each exponential is off by at most the rounding of its
argument (2^-23 of at most 30 * 1.45) and 2 ulp of exp2, a thread adds up to 130 partial sums one after the other (130 * 2^-24) and
the threads' sums meet in a tree: the sum, and with it a log-probability, is off by less than 5.2e-6 + 2.4e-7 + 7.8e-6 < SUM = 1.5e-5.
A coefficient that holds exp(lp - old) is off by that share, a softmax entry by that share of itself and its own exponential's
5.5e-6: for a gradient c * (delta - p), |c| * (delta + p) * 4e-5 bounds both with the rounding of their product.  On top comes
the rounding of the result, half a step of its type, and for 16-bit halves half of the smallest step, 2^-25."""
import math

import numpy as np
import pytest
import torch

from slayerpytorch_b200 import layer, loss

pytestmark = pytest.mark.gpu

SUM, REL = 1.5e-5, 4e-5
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def logits_of(shape, dtype, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * spread).to(dtype), gen


def want_logp(logits, action, scale=1.0):
    z = torch.log_softmax(logits.double() * scale, -1)
    return z.gather(-1, action[..., None].long())[..., 0]


def want_grad(logits, action, coef, scale=1.0):
    """(gradient, what it may be off by beside its rounding)"""
    p = torch.softmax(logits.double() * scale, -1)
    delta = torch.zeros_like(p).scatter_(-1, action[..., None].long(), 1.0)
    c = (coef * scale)[..., None]
    return c * (delta - p), c.abs() * (delta + p) * REL


def close(got, want, slack):
    assert got.shape == want.shape
    eps = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2e-38
    got = got.double().cpu()
    off = (got - want).abs()
    bound = slack + eps * (want.abs() + slack) + tiny
    assert bool((off <= bound).all()), "off by %g of the bound" % float((off / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (64, 10), (5, 31), (70, 33), (9, 257), (17, 1024), (33, 1025), (7, 4099), (3, 8193),
                                    (300, 1031), (2, 33001), (1, 66000)])
def test_log_prob_and_its_gradient(rows, V, dtype):
    x, gen = logits_of((rows, V), dtype, rows * 7 + V)
    action = torch.randint(0, V, (rows,), generator=gen)
    up = torch.randn(rows, generator=gen)
    d = x.cuda().requires_grad_()
    lp = loss.actionLogProb(d, action.cuda(), scale=0.7)
    (g,) = torch.autograd.grad(lp, [d], up.cuda())
    assert lp.dtype == torch.float32 and g.dtype == dtype
    close(lp.detach(), want_logp(x, action, 0.7), SUM)
    close(g, *want_grad(x, action, up.double(), 0.7))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [10, 900, 5003])
def test_rows_that_start_anywhere(V, dtype):
    """Rows further apart than they are long, off the 16-byte grid; entries apart; one row for all; other orders of dimensions."""
    x, gen = logits_of((4, 3, V + 5), dtype, V)
    action = torch.randint(0, V, (4, 3), generator=gen)
    up = torch.randn(4, 3, generator=gen)
    wide = x.cuda()
    for name, view, ref, act in [("shifted", wide[..., 3:V + 3], x[..., 3:V + 3], action),
                                 ("apart", wide.transpose(1, 2).contiguous().transpose(1, 2)[..., :V], x[..., :V], action),
                                 ("expanded", wide[:1, :, 1:V + 1].expand(4, 3, V), x[:1, :, 1:V + 1].expand(4, 3, V), action),
                                 ("swapped", wide.transpose(0, 1)[..., 2:V + 2], x.transpose(0, 1)[..., 2:V + 2], action.t())]:
        leaf = view.detach().requires_grad_()
        lp = loss.actionLogProb(leaf, act.cuda())
        assert lp.shape == act.shape, name
        u = up if act.shape == up.shape else up.t()
        (g,) = torch.autograd.grad(lp, [leaf], u.cuda())
        close(lp.detach(), want_logp(ref, act), SUM)
        close(g, *want_grad(ref, act, u.double()))


@pytest.mark.parametrize("V", [7, 40, 2000, 20001])
def test_values_that_are_not_finite(V):
    x, gen = logits_of((6, V), torch.float32, 3)
    action = torch.randint(1, V, (6,), generator=gen)
    x[0, :] = float("nan")                      # masked: not read
    x[1, 0] = float("-inf")                     # an entry that may not be chosen
    x[2, :] = float("-inf")                     # nothing to choose from
    x[3, 0] = float("nan")
    x[4, action[4]] = float("-inf")             # chosen all the same
    x[5, :] = 3e38                              # no difference overflows
    x[5, 0] = -3e38
    mask = torch.tensor([False, True, True, True, True, True])
    leaf = x.cuda().requires_grad_()
    lp = loss.actionLogProb(leaf, action.cuda(), mask=mask.cuda())
    (g,) = torch.autograd.grad(lp.sum(), [leaf])
    lp, g = lp.detach().cpu(), g.cpu()
    assert lp[0] == 0 and bool((g[0] == 0).all())
    want = want_logp(x[1], action[1])
    assert abs(lp[1] - want) < SUM + 2 ** -24 * abs(want) and g[1, 0] == 0 and bool(torch.isfinite(g[1]).all())
    assert torch.isnan(lp[2]) and torch.isnan(lp[3]) and bool(torch.isnan(g[3]).all())
    assert lp[4] == float("-inf") and bool(torch.isfinite(g[4]).all())
    assert abs(lp[5] + math.log(V - 1)) < SUM + 2 ** -24 * math.log(V)


@pytest.mark.parametrize("V", [5, 300, 3000])
def test_an_action_outside_makes_its_own_row_nan(V):
    x, gen = logits_of((4, V), torch.float32, 5)
    for bad in (-1, V, -2 ** 40, 2 ** 40):
        action = torch.tensor([0, bad, V - 1, 1])
        leaf = x.cuda().requires_grad_()
        lp = loss.actionLogProb(leaf, action.cuda())
        (g,) = torch.autograd.grad(lp.sum(), [leaf])
        nan_rows = torch.tensor([False, True, False, False])
        assert torch.equal(torch.isnan(lp).cpu(), nan_rows)
        assert torch.equal(torch.isnan(g).all(1).cpu(), nan_rows) and torch.equal(torch.isnan(g).any(1).cpu(), nan_rows)


# ------------------------------------------------------------------------------------------------- policy
RATIOS = [0.3, 0.7, 0.79, 0.81, 0.95, 1.0, 1.1, 1.19, 1.22, 1.27, 1.29, 2.5]       # none within 1e-2 of a border (0.8, 1.28)
CLIP = (0.2, 0.28)


def policy_case(S, L, V, dtype, seed, kl=True, masked=True):
    x, gen = logits_of((S, L, V), dtype, seed)
    action = torch.randint(0, V, (S, L), generator=gen)
    lp = want_logp(x, action, 0.9)
    old = (lp - torch.tensor(RATIOS, dtype=torch.float64)[torch.randint(0, len(RATIOS), (S, L), generator=gen)].log()).float()
    ref = (lp + 0.5 * torch.randn(S, L, generator=gen)).float() if kl else None
    adv = torch.randn(S, L, generator=gen)
    adv[0, 0] = 0.0
    mask = None
    if masked:
        mask = torch.rand(S, L, generator=gen) < 0.7
        mask[S // 2] = False                   # a sequence with nothing in it
    return x, action, old, adv, ref, mask


def policy_want(x, action, old, adv, ref, mask, kl, reduction, scale=0.9):
    """(loss, what it may be off by, coefficients)"""
    lp = want_logp(x, action, scale)
    S, L = lp.shape
    r = (lp - old.double()).exp()
    A = adv.double() if adv.shape == lp.shape else adv.double()[:, None].expand(S, L)
    lo, hi = 1 - CLIP[0], 1 + CLIP[1]
    cut = torch.where(A >= 0, r > hi, r < lo)
    per = -torch.where(cut, r.clamp(lo, hi), r) * A
    slope = torch.where(cut, torch.zeros_like(r), -r * A)
    size = r * A.abs()
    if ref is not None:
        d = ref.double() - lp
        per, slope = per + kl * (d.exp() - d - 1), slope + kl * (1 - d.exp())
        size = size + kl * (d.exp() + 1)
    keep = torch.ones(S, L, dtype=torch.float64) if mask is None else mask.double()
    if reduction == "mean":
        keep = keep / max(1.0, float(keep.sum()))
    elif reduction == "sequence":
        keep = keep / keep.sum(1, keepdim=True).clamp(min=1) / S
    # the slope by lp is at most `size`, so an error of SUM in lp moves the loss by SUM * size
    return (per * keep).sum(), (size * keep).sum() * SUM, slope * keep, size * keep


@pytest.mark.parametrize("reduction", ["sum", "mean", "sequence"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,L,V,kl,masked", [(1, 1, 2, False, False), (16, 4, 10, True, True), (6, 1, 33, False, True), (5, 9, 700, True, True),
                                             (3, 7, 1030, True, False), (4, 5, 5001, True, True), (2, 3, 40003, True, True)])
def test_policy_loss_and_gradient(S, L, V, kl, masked, dtype, reduction):
    x, action, old, adv, ref, mask = policy_case(S, L, V, dtype, S + V, kl, masked)
    leaf = x.cuda().requires_grad_()
    dev = [t if t is None else t.cuda() for t in (action, old, adv, ref, mask)]
    got, lp = loss.policyLoss(leaf, dev[0], dev[1], dev[2], refLogProb=dev[3], mask=dev[4], clip=CLIP, klCoef=0.3 if kl else 0.0, scale=0.9,
                              reduction=reduction, returnLogProb=True)
    value, slack, coef, size = policy_want(x, action, old, adv, ref, mask, 0.3, reduction)
    assert got.dtype == torch.float32 and got.shape == () and lp.shape == (S, L)
    assert abs(float(got.detach()) - float(value.detach())) <= float(slack) + 2 ** -24 * abs(float(value.detach())) + 1e-30
    keep = torch.ones(S, L, dtype=torch.bool) if mask is None else mask
    close(lp, torch.where(keep, want_logp(x, action, 0.9), 0.0), SUM)
    (g,) = torch.autograd.grad(got, [leaf], retain_graph=True)
    grad, spare = want_grad(x, action, coef, 0.9)
    # the coefficient's own error is SUM of what it is made of
    spare = spare + 0.9 * (size * SUM)[..., None] * (grad / torch.where(coef == 0, 1.0, coef * 0.9)[..., None]).abs()
    close(g, grad, spare)
    assert bool((g[~keep.cuda()] == 0).all())
    # a later backward pass, and one whose upstream gradient is not one
    (again,) = torch.autograd.grad(got, [leaf], retain_graph=True)
    assert torch.equal(again, g)
    (scaled,) = torch.autograd.grad(got * 8.0, [leaf])
    close(scaled, grad * 8.0, spare * 8.0)


@pytest.mark.parametrize("dtype,V", [(torch.float32, 9001), (torch.float32, 70001), (torch.bfloat16, 20003), (torch.float16, 120001), (torch.bfloat16, 40000)])
@pytest.mark.parametrize("masked", [True, False])
def test_policy_many_long_rows(dtype, V, masked):
    """Enough rows for the walk over them, in one CTA and in clusters, rows that start anywhere."""
    S, L = 40, 9
    x, action, old, adv, ref, mask = policy_case(S, L, V, dtype, V, True, masked)
    x64 = x.cuda().double()
    leaf = x.cuda().requires_grad_()
    dev = [t if t is None else t.cuda() for t in (action, old, adv, ref, mask)]
    for want in (True, False):
        with torch.set_grad_enabled(want):
            got, lp = loss.policyLoss(leaf, dev[0], dev[1], dev[2], refLogProb=dev[3], mask=dev[4], clip=CLIP, klCoef=0.3, scale=0.9, reduction="mean",
                                      returnLogProb=True)
        value, slack, coef, size = policy_want(x64, dev[0], dev[1], dev[2], dev[3], dev[4] if masked else torch.ones(S, L, device="cuda").bool(), 0.3, "mean")
        assert abs(float(got.detach()) - float(value)) <= float(slack) + 2 ** -24 * abs(float(value)) + 1e-30
        keep = torch.ones(S, L, dtype=torch.bool) if mask is None else mask
        close(lp, torch.where(keep, want_logp(x64, dev[0], 0.9).cpu(), 0.0), SUM)
    got = loss.policyLoss(leaf, dev[0], dev[1], dev[2], refLogProb=dev[3], mask=dev[4], clip=CLIP, klCoef=0.3, scale=0.9, reduction="mean")
    (g,) = torch.autograd.grad(got, [leaf], retain_graph=True)
    (again,) = torch.autograd.grad(got, [leaf])
    assert torch.equal(g, again)
    for s in range(0, S, 13):
        grad, spare = want_grad(x64[s], dev[0][s], coef[s], 0.9)
        spare = spare + 0.9 * (size[s] * SUM)[..., None] * (grad / torch.where(coef[s] == 0, 1.0, coef[s] * 0.9)[..., None]).abs()
        close(g[s], grad.cpu(), spare.cpu())


@pytest.mark.parametrize("V", [12, 3001])
def test_policy_advantage_of_a_whole_sequence_and_first_backward_scaled(V):
    x, action, old, adv, ref, mask = policy_case(6, 5, V, torch.float32, 11)
    leaf = x.cuda().requires_grad_()
    args = dict(refLogProb=ref.cuda(), mask=mask.cuda(), clip=CLIP, klCoef=0.3, scale=0.9, reduction="sequence")
    by_row = loss.policyLoss(leaf, action.cuda(), old.cuda(), adv[:, :1].expand(6, 5).cuda(), **args)
    by_seq = loss.policyLoss(leaf, action.int().cuda(), old.cuda(), adv[:, 0].cuda(), **args)
    assert torch.equal(by_row, by_seq)
    (g,) = torch.autograd.grad(by_row, [leaf])
    (g3,) = torch.autograd.grad(by_seq * 3.0, [leaf])           # the gradient that the forward pass left is not used
    value, slack, coef, size = policy_want(x, action, old, adv[:, 0], ref, mask, 0.3, "sequence")
    grad, spare = want_grad(x, action, coef, 0.9)
    spare = spare + 0.9 * (size * SUM)[..., None] * (grad / torch.where(coef == 0, 1.0, coef * 0.9)[..., None]).abs()
    close(g, grad, spare)
    close(g3, 3 * grad, 3 * spare)


def test_policy_gradient_against_differences():
    """The kernels' gradient against differences of the kernels' own loss, 64 terms of order one: a step of 2^-6 moves a
    log-probability by up to 2^-6, the third derivative adds 2^-12 / 6 of the size, the fp32 loss 2^-24 * 64 / 2^-6."""
    x, action, old, adv, ref, _ = policy_case(4, 4, 9, torch.float32, 21, masked=False)
    lp = want_logp(x, action, 0.9)
    old = (lp - 0.05 * torch.sign(adv)).float()                # inside the clip range, so that the loss is smooth
    args = dict(refLogProb=ref.cuda(), clip=CLIP, klCoef=0.3, scale=0.9)
    leaf = x.cuda().requires_grad_()
    (g,) = torch.autograd.grad(loss.policyLoss(leaf, action.cuda(), old.cuda(), adv.cuda(), **args), [leaf])
    h = 2.0 ** -6
    for s, l, v in [(0, 0, 0), (1, 2, 3), (3, 3, 8), (2, 1, int(action[2, 1]))]:
        values = []
        for sign in (1, -1):
            y = x.clone()
            y[s, l, v] += sign * h
            values.append(float(loss.policyLoss(y.cuda(), action.cuda(), old.cuda(), adv.cuda(), **args)))
        size = float(adv[s, l].abs()) * 2 + 2
        assert abs((values[0] - values[1]) / (2 * h) - float(g[s, l, v])) < size * h * h + 64 * 2 ** -24 / h


def test_policy_rows_that_are_all_masked_or_missing():
    for reduction in ("sum", "mean", "sequence"):
        for S, L in ((3, 4), (0, 4), (3, 0)):
            leaf = torch.full((S, L, 50), float("nan"), device="cuda", requires_grad=True)
            z = torch.zeros(S, L, device="cuda")
            got = loss.policyLoss(leaf, z.long(), z, z, mask=z.bool(), reduction=reduction)
            (g,) = torch.autograd.grad(got, [leaf])
            assert float(got.detach()) == 0.0 and bool((g == 0).all()) and g.shape == leaf.shape
    lp = loss.actionLogProb(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"))
    assert lp.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_second_derivative_is_refused(dtype):
    x = torch.randn(6, 4, 9, device="cuda").to(dtype).requires_grad_()
    a = torch.randint(0, 9, (6, 4), device="cuda")
    zero = torch.zeros(6, 4, device="cuda")
    for make in (lambda: loss.actionLogProb(x, a).sum(), lambda: loss.policyLoss(x, a, zero - 2, zero + 1),
                 lambda: loss.preferenceLoss(x, a, zero[:, 0])):
        plain, = torch.autograd.grad(make(), x)
        g, = torch.autograd.grad(make(), x, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="first derivatives only"):
            g.float().square().sum().backward()


def test_policy_without_gradients_writes_none():
    x, action, old, adv, ref, mask = policy_case(3, 4, 2000, torch.bfloat16, 2)
    leaf = x.cuda().requires_grad_()
    with torch.no_grad():
        a = loss.policyLoss(leaf, action.cuda(), old.cuda(), adv.cuda(), mask=mask.cuda(), scale=0.9)
    assert not a.requires_grad
    b = loss.policyLoss(leaf, action.cuda(), old.cuda(), adv.cuda(), mask=mask.cuda(), scale=0.9)
    assert torch.equal(a, b.detach())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [11, 2049])
def test_policy_in_a_graph(V, dtype):
    """A captured step replays on new data.  (An eager graph of the same leaf must not live meanwhile: autograd ties a leaf's node to
    the stream it was made on, and refuses to capture across it, whatever the operators.)"""
    x, action, old, adv, ref, mask = policy_case(4, 3, V, dtype, 31)
    leaf = x.cuda().requires_grad_()
    dev = [t.cuda() for t in (action, old, adv, ref, mask)]

    def step():
        value = loss.policyLoss(leaf, dev[0], dev[1], dev[2], refLogProb=dev[3], mask=dev[4], clip=CLIP, klCoef=0.3, scale=0.9, reduction="mean")
        return value, torch.autograd.grad(value, [leaf], retain_graph=True)[0]

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        value, g = step()
    y, *new = policy_case(4, 3, V, dtype, 32)
    with torch.no_grad():
        leaf.copy_(y.cuda())
    for d, n in zip(dev, new):
        d.copy_(n.cuda())
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want_value, want = step()
    assert torch.equal(value, want_value) and torch.equal(g, want)


def test_policy_backward_captured_alone_forms_its_gradient():
    x, action, old, adv, ref, mask = policy_case(4, 3, 1500, torch.float32, 41)
    leaf = x.cuda().requires_grad_()
    dev = [t.cuda() for t in (action, old, adv)]
    one = torch.ones((), device="cuda")
    side = torch.cuda.Stream()              # autograd runs a backward pass on the stream of its forward pass
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (want,) = torch.autograd.grad(loss.policyLoss(leaf, *dev, clip=CLIP, scale=0.9), [leaf])
        value = loss.policyLoss(leaf, *dev, clip=CLIP, scale=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (g,) = torch.autograd.grad(value, [leaf], one, retain_graph=True)
    graph.replay()
    torch.cuda.synchronize()
    g.zero_()                                   # the user's own buffer by now
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want)


def test_policy_on_another_stream():
    x, action, old, adv, ref, mask = policy_case(8, 16, 4000, torch.float32, 51)
    leaf = x.cuda().requires_grad_()
    dev = [t.cuda() for t in (action, old, adv)]
    want = loss.policyLoss(leaf, *dev, clip=CLIP, scale=0.9)
    (wg,) = torch.autograd.grad(want, [leaf])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            v = loss.policyLoss(leaf, *dev, clip=CLIP, scale=0.9)
            got.append((v, torch.autograd.grad(v, [leaf])[0]))
    torch.cuda.synchronize()
    for v, g in got:
        assert torch.equal(v, want) and torch.equal(g, wg)


# --------------------------------------------------------------------------------------------- preference
def preference_want(x, action, ref, pairs, mask, beta, smoothing, reduction, scale=0.9):
    lp = want_logp(x, action, scale)
    keep = torch.ones_like(lp) if mask is None else mask.double()
    lp = torch.where(keep > 0, lp, 0.0)
    S, L = lp.shape
    m = lp.sum(1) - ref.double()
    h = beta * (m[pairs[:, 0]] - m[pairs[:, 1]])
    each = -(1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)
    share = 1.0 if reduction == "sum" or len(h) == 0 else 1.0 / len(h)
    slope = share * beta * (torch.sigmoid(h) - (1 - smoothing))
    coef = torch.zeros(S, dtype=torch.float64).index_add_(0, pairs[:, 0], slope).index_add_(0, pairs[:, 1], -slope)
    # lp is off by SUM and its own rounding, a margin by L of those; the loss's slope by a margin is at most beta, a slope's at most beta^2 / 4
    dm = L * (SUM + 2 ** -24 * float(lp.abs().max() if lp.numel() else 0))
    many = torch.zeros(S, dtype=torch.float64).index_add_(0, pairs.reshape(-1), torch.ones(2 * len(pairs), dtype=torch.float64))
    return each.sum() * share, 2 * beta * dm * share * len(h), coef[:, None] * keep, (many * share * beta * beta / 2 * dm)[:, None] * keep


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,L,V,masked", [(2, 1, 2, False), (32, 20, 11, True), (6, 5, 600, True), (5, 3, 2050, False), (700, 2, 5, True)])
def test_preference_loss_and_gradient(S, L, V, masked, dtype, reduction):
    x, gen = logits_of((S, L, V), dtype, S * L + V)
    action = torch.randint(0, V, (S, L), generator=gen)
    mask = None
    if masked:
        mask = torch.arange(L)[None] < torch.randint(0, L + 1, (S, 1), generator=gen)
        mask[0] = False
    lp = want_logp(x, action, 0.9)
    ref = (lp.sum(1) + 2 * torch.randn(S, generator=gen)).float()
    pairs = torch.cat([torch.randint(0, S, (3 + S // 2, 2), generator=gen), torch.tensor([[0, 1], [0, 1], [1, 1]])])
    leaf = x.cuda().requires_grad_()
    got = loss.preferenceLoss(leaf, action.cuda(), ref.cuda(), pairs=pairs.cuda(), mask=None if mask is None else mask.cuda(), beta=0.4,
                              labelSmoothing=0.2, scale=0.9, reduction=reduction)
    value, slack, coef, spare_coef = preference_want(x, action, ref, pairs, mask, 0.4, 0.2, reduction)
    assert abs(float(got.detach()) - float(value.detach())) <= slack + 2 ** -23 * abs(float(value.detach()))
    for up in (1.0, 0.25):
        (g,) = torch.autograd.grad(got * up, [leaf], retain_graph=True)
        grad, spare = want_grad(x, action, coef, 0.9)
        p = torch.softmax(x.double() * 0.9, -1)
        spare = spare + 0.9 * spare_coef[..., None] * (p + torch.zeros_like(p).scatter_(-1, action[..., None], 1.0))
        close(g, up * grad, up * spare)


def test_preference_default_pairs_extremes_and_bad_indices():
    S, L, V = 6, 4, 20
    x, gen = logits_of((S, L, V), torch.float32, 8)
    action = torch.randint(0, V, (S, L), generator=gen)
    leaf = x.cuda().requires_grad_()
    ref = torch.zeros(S)
    halves = torch.stack([torch.arange(3), torch.arange(3) + 3], 1)
    a = loss.preferenceLoss(leaf, action.cuda(), ref.cuda())
    b = loss.preferenceLoss(leaf, action.cuda(), ref.cuda(), pairs=halves.int().cuda())
    assert torch.equal(a, b)
    # margins far apart: the loss is linear there, and its gradient neither overflows nor vanishes
    for sign in (1.0, -1.0):
        far = torch.tensor([sign * 1e6] * 3 + [0.0] * 3)
        v = loss.preferenceLoss(leaf, action.cuda(), far.cuda())
        (g,) = torch.autograd.grad(v, [leaf])
        assert abs(float(v.detach()) - (3e5 if sign > 0 else 0.0)) < 20 and bool(torch.isfinite(g).all())
        assert bool((g != 0).any()) == (sign > 0)
    for bad in ([[0, 6]], [[-1, 2]], [[0, 1], [2 ** 40, 2]]):
        v = loss.preferenceLoss(leaf, action.cuda(), ref.cuda(), pairs=torch.tensor(bad).cuda())
        (g,) = torch.autograd.grad(v, [leaf])
        assert torch.isnan(v)
        hit = {i for p in bad if any(not 0 <= q < S for q in p) for i in p if 0 <= i < S}
        assert {int(i) for i in torch.isnan(g).any(2).any(1).nonzero()} == hit
    none = loss.preferenceLoss(leaf, action.cuda(), ref.cuda(), pairs=torch.empty(0, 2, dtype=torch.long).cuda(), reduction="mean")
    (g,) = torch.autograd.grad(none, [leaf])
    assert float(none) == 0.0 and bool((g == 0).all())
    empty = torch.zeros(2, 0, 5, device="cuda", requires_grad=True)
    v = loss.preferenceLoss(empty, torch.zeros(2, 0, dtype=torch.long, device="cuda"), torch.zeros(2).cuda())
    (g,) = torch.autograd.grad(v, [empty])
    assert abs(float(v.detach()) - math.log(2)) < 1e-6 and g.shape == empty.shape


# --------------------------------------------------------------------------------------- from spike counts
def descriptor(kind, **more):
    return {"neuron": {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1},
            "simulation": {"Ts": 1.0, "tSample": 50},
            "training": {"error": {"type": kind, "tgtSpikeRegion": {"start": 5, "stop": 45}, "countScale": 0.25, **more}}}


def test_spike_loss_policy_and_preference():
    gen = torch.Generator().manual_seed(4)
    spikes = (torch.rand(12, 7, 1, 1, 50, generator=gen) < 0.2).float()
    action = torch.randint(0, 7, (12,), generator=gen)
    counts = spikes[..., 5:45].sum(-1).reshape(12, 7)
    lp = want_logp(counts, action, 0.25)
    net = loss.spikeLoss(descriptor("Policy", clip=CLIP, klCoef=0.3)).cuda()
    leaf = spikes.cuda().requires_grad_()
    close(net.actionLogProb(leaf, action.cuda()).detach(), lp, SUM)
    old, ref, adv = (lp + 0.1).float(), (lp - 0.2).float(), torch.randn(12, generator=gen)
    got = net.policy(leaf, action.cuda(), old.cuda(), adv.cuda(), refLogProb=ref.cuda())
    value, slack, coef, size = policy_want(counts[:, None], action[:, None], old[:, None], adv[:, None], ref[:, None], None, 0.3, "sum", 0.25)
    assert abs(float(got.detach()) - float(value.detach())) <= float(slack) + 2 ** -24 * abs(float(value.detach()))
    got.backward()
    grad, spare = want_grad(counts, action, coef[:, 0], 0.25)
    spare = spare + 0.25 * (size * SUM)
    want = torch.zeros(12, 7, 1, 1, 50, dtype=torch.float64)
    want[..., 5:45] = grad.reshape(12, 7, 1, 1, 1)
    close(leaf.grad, want, spare.reshape(12, 7, 1, 1, 1).expand_as(want))

    pref = loss.spikeLoss(descriptor("Preference", beta=0.4)).cuda()
    two = action.reshape(4, 3)
    refs = torch.randn(4, generator=gen)
    pairs = torch.tensor([[0, 2], [1, 3]])
    got = pref.preference(leaf, two.cuda(), refs.cuda())
    value, slack, _, _ = preference_want(counts.reshape(4, 3, 7), two, refs, pairs, None, 0.4, 0.0, "sum", 0.25)
    assert abs(float(got.detach()) - float(value.detach())) <= slack + 2 ** -23 * abs(float(value.detach()))


def test_a_spiking_network_is_trained_by_reward():
    """The layers, the log-probabilities of the choices made, the loss and its gradient in the weights, as they are used together."""
    d = descriptor("Policy")
    net = layer.spikeLayer(d["neuron"], d["simulation"]).cuda()
    torch.manual_seed(3)
    dense = net.dense(20, 5, weightScale=10).cuda()
    error = loss.spikeLoss(d).cuda()
    x = (torch.rand(16, 20, 1, 1, 50, device="cuda") < 0.3).float()
    spikes = net.spike(dense(net.psp(x)))
    with torch.no_grad():
        label = loss.spikeClassifier.getClass(spikes, host=False)
        old = error.actionLogProb(spikes, label)
    value = error.policy(spikes, label, old, torch.ones(16, device="cuda"))
    assert abs(float(value) + 16) < 16 * SUM            # ratio 1, advantage 1
    value.backward()
    assert bool(torch.isfinite(dense.weight.grad).all()) and float(dense.weight.grad.abs().max()) > 0


def test_refusals_on_the_device():
    x = torch.zeros(4, 6, device="cuda")
    a = torch.zeros(4, dtype=torch.long, device="cuda")
    z = torch.zeros(4, device="cuda")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        loss.actionLogProb(x.double(), a)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        loss.actionLogProb(x, a.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        loss.policyLoss(x, a, z.cpu(), z)
    leaf = x.clone().requires_grad_()
    value = loss.policyLoss(leaf, a, z, z + 1)
    (g,) = torch.autograd.grad(value, [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|differentiate"):
        torch.autograd.grad(g.sum(), [leaf])
