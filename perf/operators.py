"""The learning operators of the package, as cases that can be timed and compared with their plain forms.

A network that answers with choices - the spike counts of its output neurons, or the logits of a large vocabulary -
is trained here by what its choices were worth, and its weight matrices by orthogonalised updates:

``logprob``     the log-probability of the chosen entry of each row of logits, and its gradient
``policy``      the clipped policy loss with a KL term over rows of logits, and its gradient
``preference``  the loss of paired sequences (which of two is preferred), and its gradient
``orthogonal``  a matrix, or a stack of them, made near orthogonal by Newton-Schulz products
``muon``        one optimiser step of a network: momentum, orthogonalisation and update of each weight

Logits are ``[S, L, V]``: S sequences (episodes) of L choices among V entries.  Weights are given by their shapes, as the
layers hold them: ``[out, in, kh, kw, 1]`` of a convolution is a matrix of ``out`` rows.
"""
import math

import torch

own = False

#: Newton-Schulz coefficients: the quintic whose slope at zero is as steep as it can be with every singular value ending near one.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
CLIP, KL, BETA, SMOOTHING = (0.2, 0.28), 0.04, 0.1, 0.1
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the 2-16-32-64-10 spiking CNN's weights, one step: an experiment's network, bound by latency
        _muon("muon_cnn", "16x2x5x5x1 32x16x3x3x1 64x32x3x3x1 10x64x8x8x1", "float32"),
        # the 2312-512-10 spiking classifier's weights, one step
        _muon("muon_mlp", "512x2312x1x1x1 10x512x1x1x1", "float32"),
        # a wide network's square and rectangular weights in 32 bits: the largest work of all
        _muon("muon_large", "4096x4096 1024x4096", "float32"),
        # a stack of equal weights in 16 bits, sizes that no tile divides
        _orthogonal("orthogonal_odd", 6, 1023, 2049, "bfloat16"),
        # one tall matrix in 32 bits
        _orthogonal("orthogonal_tall", 1, 2000, 333, "float32"),
        # a batch of a ten-class spiking classifier trained by reward: the logits are spike counts
        _policy("policy_counts", 64, 1, 10, "float32", "sum", False, False, 0.2),
        # answers of a large vocabulary, ragged lengths, with the KL term
        _policy("policy_tokens", 8, 512, 32768, "bfloat16", "sequence", True, True, 1.0),
        # an odd vocabulary in 32 bits: rows that start anywhere
        _policy("policy_odd", 5, 301, 50021, "float32", "mean", True, True, 1.0),
        # pairs of short episodes of a spiking network with eleven gestures to choose from
        _preference("preference_counts", 32, 20, 11, "float32", True, 0.2),
        # pairs of long answers
        _preference("preference_tokens", 16, 256, 32000, "bfloat16", True, 1.0),
        # the old log-probabilities of a few next tokens: one row for each request
        _logprob("logprob_one", 8, 1, 131072, "bfloat16", False, False, 1.0),
        # log-probabilities that something else is made of, with their gradient
        _logprob("logprob_train", 16, 100, 8191, "float16", True, True, 1.0),
    ]


def _muon(name, shapes, dtype):
    return _named(name, {"kind": "muon", "shapes": shapes, "dtype": dtype})


def _orthogonal(name, B, R, C, dtype):
    return _named(name, {"kind": "orthogonal", "B": B, "R": R, "C": C, "dtype": dtype})


def _policy(name, S, L, V, dtype, reduction, kl, masked, scale):
    return _named(name, {"kind": "policy", "S": S, "L": L, "V": V, "dtype": dtype, "reduction": reduction, "kl": kl, "masked": masked,
                         "scale": scale})


def _preference(name, S, L, V, dtype, masked, scale):
    return _named(name, {"kind": "preference", "S": S, "L": L, "V": V, "dtype": dtype, "masked": masked, "scale": scale})


def _logprob(name, S, L, V, dtype, masked, grad, scale):
    return _named(name, {"kind": "logprob", "S": S, "L": L, "V": V, "dtype": dtype, "masked": masked, "grad": grad, "scale": scale})


def _named(name, case):
    return {"name": name, **case} if name else case


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["muon", "muon", "muon", "orthogonal", "orthogonal", "policy", "policy", "policy", "preference", "preference", "logprob"])
    dtype = rng.choice(list(TYPES))
    if kind in ("muon", "orthogonal"):
        most = 1e12 if rng.random() < 0.3 else 5e10
        R, C, count = log(4, 4096), log(4, 8192), log(1, 8)
        while True:
            case = _orthogonal(None, count, R, C, dtype)
            if kind == "muon":
                sides = [(max(1, int(R * 2 ** -rng.randint(0, 2))), max(1, int(C * 2 ** -rng.randint(0, 2)))) for _ in range(count)]
                case = _muon(None, " ".join("%dx%d" % s for s in sides), dtype)
            if work(case)["flops"] <= most:
                return case
            R, C, count = (R + 1) // 2, (C + 1) // 2, (count + 1) // 2
    V = log(2, 150000)
    rows = min(log(1, 16384), 10 ** 8 // V + 1)
    S = min(rows, log(1, 64))
    L = max(1, rows // S)
    masked, scale = rng.random() < 0.6, rng.choice([1.0, 1.0, 0.2])
    if kind == "policy":
        return _policy(None, S, L, V, dtype, rng.choice(["sum", "mean", "sequence"]), rng.random() < 0.7, masked, scale)
    if kind == "preference":
        return _preference(None, S + S % 2, L, V, dtype, masked, scale)
    return _logprob(None, S, L, V, dtype, masked, rng.random() < 0.5, scale)


# ------------------------------------------------------------------------------------------------ inputs
def _gradient(shape, gen):
    """A weight's gradient as training gives it: a few strong directions over noise."""
    R, C = shape[0], math.prod(shape[1:])
    dev = torch.device("cuda")
    k = min(8, R, C)
    u = torch.empty((R, k), device=dev).normal_(generator=gen)
    v = torch.empty((k, C), device=dev).normal_(generator=gen)
    strength = 2.0 ** -torch.arange(k, device=dev, dtype=torch.float32)
    return ((u * strength) @ v + torch.empty((R, C), device=dev).normal_(generator=gen)).mul_(1e-3).reshape(shape)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["kind"] == "orthogonal":
        state["matrix"] = torch.stack([_gradient((case["R"], case["C"]), gen) for _ in range(case["B"])]).to(dtype)
        return state
    if case["kind"] == "muon":
        shapes = [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()]
        state["weights"] = [torch.empty(s, device=dev).normal_(generator=gen).div_(math.sqrt(math.prod(s[1:]))).to(dtype) for s in shapes]
        state["grads"] = [_gradient(s, gen).to(dtype) for s in shapes]
        state["momenta"] = [_gradient(s, gen).mul_(8.0) for s in shapes]
        return state
    S, L, V, scale = case["S"], case["L"], case["V"], case["scale"]
    normal = lambda *shape: torch.empty(shape, device=dev).normal_(generator=gen)  # noqa: E731
    if scale == 1.0:
        logits = normal(S, L, V).mul_(2.0)
    else:       # spike counts
        logits = normal(S, L, V).mul_(6.0).add_(12.0).round_().clamp_(min=0.0)
    action = torch.randint(0, V, (S, L), device=dev, generator=gen)
    # a choice that the network finds likely
    logits.scatter_add_(2, action[..., None], normal(S, L, 1).abs_().add_(0.75 * math.log(V)).div_(scale))
    if scale != 1.0:
        logits.round_()
    logits = logits.to(dtype)
    state["action"] = action
    state["mask"] = None
    if case["masked"]:      # padded behind each sequence's own length; one now and then is empty
        length = torch.randint(0, L + 1, (S, 1), device=dev, generator=gen)
        length[: (S + 1) // 2] = torch.clamp(length[: (S + 1) // 2], min=(L + 1) // 2)
        state["mask"] = torch.arange(L, device=dev)[None] < length
    if case["kind"] == "logprob":
        state["logits"] = logits.requires_grad_(case["grad"])
        state["upstream"] = normal(S, L)
        return state
    with torch.no_grad():
        z = logits.float().mul_(scale)
        lp = z.gather(2, action[..., None])[..., 0] - z.logsumexp(2)
        del z
    if case["kind"] == "policy":
        state["old"] = lp + 0.2 * normal(S, L)
        state["ref"] = lp + 0.3 * normal(S, L) if case["kl"] else None
        state["advantage"] = normal(S, 1).expand(S, L).contiguous() if case["reduction"] == "sequence" else normal(S, L)
    else:
        kept = lp if state["mask"] is None else lp * state["mask"]
        state["ref"] = kept.sum(1) + 3.0 * normal(S)
        # each sequence in one pair, and some of them in more
        pairs = torch.randperm(S, device=dev, generator=gen).reshape(-1, 2)
        extra = torch.randint(0, S, (S // 4, 1), device=dev, generator=gen)
        state["pairs"] = torch.cat([pairs, torch.cat([extra, (extra + 1 + S // 2) % S], 1)]) if S > 4 else pairs
    state["logits"] = logits.requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------- the plain forms
def _plain_log_prob(state):
    case, x = state["case"], state["logits"]
    z = x.float() * case["scale"]
    top = z.detach().amax(2, keepdim=True)
    total = torch.exp(z - top).sum(2, dtype=torch.float64)
    # what is next to a border of the clip range is decided in 64 bits
    lp = (z.gather(2, state["action"][..., None]) - top)[..., 0].double() - torch.log(total)
    return lp if state["mask"] is None else torch.where(state["mask"], lp, 0.0)


def _plain_policy(state):
    case, mask = state["case"], state["mask"]
    lp = _plain_log_prob(state)
    ratio = torch.exp(lp - state["old"].double())
    gain = state["advantage"].double()
    per = -torch.minimum(ratio * gain, torch.clamp(ratio, 1.0 - CLIP[0], 1.0 + CLIP[1]) * gain)
    if state["ref"] is not None:
        away = state["ref"].double() - lp
        per = per + KL * (torch.exp(away) - away - 1.0)
    if mask is None:
        mask = torch.ones_like(per, dtype=torch.bool)
    per = torch.where(mask, per, 0.0)
    if case["reduction"] == "sum":
        return per.sum().float()
    if case["reduction"] == "mean":
        return (per.sum() / mask.sum().clamp(min=1)).float()
    return (per.sum(1) / mask.sum(1).clamp(min=1)).mean().float()


def _plain_preference(state):
    margin = _plain_log_prob(state).sum(1) - state["ref"].double()
    h = BETA * (margin[state["pairs"][:, 0]] - margin[state["pairs"][:, 1]])
    tail = torch.log1p(torch.exp(-h.abs()))
    zero = torch.zeros_like(h)
    per = (1.0 - SMOOTHING) * (torch.maximum(-h, zero) + tail) + SMOOTHING * (torch.maximum(h, zero) + tail)
    return per.mean().float()


def _plain_orthogonalize(matrix):
    a, b, c = COEFFICIENTS
    x = matrix.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / (norm + EPS).float()
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain_muon(state):
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        g = g.float()
        m.mul_(MOMENTUM).add_(g)
        rows, cols = w.shape[0], math.prod(w.shape[1:])
        o = _plain_orthogonalize((g + MOMENTUM * m).reshape(rows, cols)).reshape(w.shape)
        step = LR * math.sqrt(max(1.0, rows / cols))
        w.copy_(w.float() * (1.0 - LR * DECAY) - step * o)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "muon":
        if own:
            from slayerpytorch_b200.optim import muonStep
            muonStep(state["weights"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM, weightDecay=DECAY)
        else:
            _plain_muon(state)
        return [*state["weights"], *state["momenta"]]
    if kind == "orthogonal":
        if own:
            from slayerpytorch_b200.optim import orthogonalize
            return orthogonalize(state["matrix"])
        return _plain_orthogonalize(state["matrix"]).to(state["matrix"].dtype)
    if kind == "logprob":
        with torch.set_grad_enabled(case["grad"]):
            if own:
                from slayerpytorch_b200.loss import actionLogProb
                lp = actionLogProb(state["logits"], state["action"], mask=state["mask"], scale=case["scale"])
            else:
                lp = _plain_log_prob(state).float()
        if not case["grad"]:
            return lp
        return [lp.detach(), *torch.autograd.grad(lp, [state["logits"]], state["upstream"])]
    if kind == "policy":
        if own:
            from slayerpytorch_b200.loss import policyLoss
            loss = policyLoss(state["logits"], state["action"], state["old"], state["advantage"], refLogProb=state["ref"], mask=state["mask"],
                              clip=CLIP, klCoef=KL if case["kl"] else 0.0, scale=case["scale"], reduction=case["reduction"])
        else:
            loss = _plain_policy(state)
    elif own:
        from slayerpytorch_b200.loss import preferenceLoss
        loss = preferenceLoss(state["logits"], state["action"], state["ref"], pairs=state["pairs"], mask=state["mask"], beta=BETA,
                              labelSmoothing=SMOOTHING, scale=case["scale"], reduction="mean")
    else:
        loss = _plain_preference(state)
    return [loss.detach(), *torch.autograd.grad(loss, [state["logits"]])]


def work(case):
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    if case["kind"] in ("muon", "orthogonal"):
        if case["kind"] == "orthogonal":
            sides, each = [(case["R"], case["C"])] * case["B"], 2 * size
        else:
            shapes = [[int(n) for n in s.split("x")] for s in case["shapes"].split()]
            sides, each = [(s[0], math.prod(s[1:])) for s in shapes], 3 * size + 8
        total = {"bytes": 0, "flops": 0}
        for r, c in sides:
            m, n = min(r, c), max(r, c)
            total["bytes"] += each * m * n
            # the Gram matrix and its square are symmetric: half of each is computed
            total["flops"] += STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        return total
    rows, V = case["S"] * case["L"], case["V"]
    grad = case["kind"] != "logprob" or case["grad"]
    return {"bytes": rows * V * size * (2 if grad else 1) + 24 * rows, "flops": rows * V * (8 if grad else 4)}


# ---------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_gradient(state, coefficient):
    """coefficient[s, l] * d log-probability / d logits, a sequence at a time."""
    case = state["case"]
    grad = torch.empty(state["logits"].shape, dtype=torch.float64, device="cuda")
    for s in range(case["S"]):
        soft = torch.softmax(state["logits"][s].detach().double() * case["scale"], -1)
        grad[s] = -case["scale"] * coefficient[s][:, None] * soft
        grad[s].scatter_add_(1, state["action"][s][:, None], case["scale"] * coefficient[s][:, None])
    return grad


def _exact_loss(state):
    case, kind = state["case"], state["case"]["kind"]
    S, L = case["S"], case["L"]
    kept = torch.ones((S, L), dtype=torch.float64, device="cuda") if state["mask"] is None else state["mask"].double()
    lp = torch.empty((S, L), dtype=torch.float64, device="cuda")
    for s in range(S):
        z = torch.log_softmax(state["logits"][s].detach().double() * case["scale"], -1)
        lp[s] = z.gather(1, state["action"][s][:, None])[:, 0] * kept[s]
    if kind == "logprob":
        return [lp, _exact_gradient(state, kept * state["upstream"].double())] if case["grad"] else lp
    if kind == "policy":
        old, gain = state["old"].double(), state["advantage"].double()
        ratio = (lp - old).exp()
        low, high = 1.0 - CLIP[0], 1.0 + CLIP[1]
        bound = torch.where(gain >= 0, torch.full_like(ratio, high), torch.full_like(ratio, low))
        cut = torch.where(gain >= 0, ratio > high, ratio < low)
        per, slope = -torch.where(cut, bound, ratio) * gain, -torch.where(cut, torch.zeros_like(ratio), ratio) * gain
        if state["ref"] is not None:
            away = state["ref"].double() - lp
            per, slope = per + KL * (away.expm1() - away), slope - KL * away.expm1()
        if case["reduction"] == "sum":
            share = kept
        elif case["reduction"] == "mean":
            share = kept / kept.sum().clamp(min=1.0)
        else:
            share = kept / (kept.sum(1, keepdim=True).clamp(min=1.0) * S)
        return [(share * per).sum(), _exact_gradient(state, share * slope)]
    margin = lp.sum(1) - state["ref"].double()
    first, second = state["pairs"].T
    h = BETA * (margin[first] - margin[second])
    loss = -((1.0 - SMOOTHING) * torch.nn.functional.logsigmoid(h) + SMOOTHING * torch.nn.functional.logsigmoid(-h)).mean()
    slope = BETA * (torch.sigmoid(h) - (1.0 - SMOOTHING)) / len(h)
    by_sequence = torch.zeros(S, dtype=torch.float64, device="cuda").index_add_(0, first, slope).index_add_(0, second, -slope)
    return [loss, _exact_gradient(state, kept * by_sequence[:, None])]


def _exact_orthogonal(x):
    a, b, c = COEFFICIENTS
    x = x.double()
    x = x / (torch.linalg.vector_norm(x) + EPS)
    eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        if x.shape[0] > x.shape[1]:
            gram = x.T @ x
            x = x @ (a * eye + b * gram + c * gram @ gram)
        else:
            gram = x @ x.T
            x = (a * eye + b * gram + c * gram @ gram) @ x
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "orthogonal":
        return torch.stack([_exact_orthogonal(x) for x in state["matrix"]])
    if case["kind"] == "muon":
        momenta = [MOMENTUM * m.double() + g.double() for m, g in zip(state["momenta"], state["grads"])]
        weights = []
        for w, g, m in zip(state["weights"], state["grads"], momenta):
            o = _exact_orthogonal((g.double() + MOMENTUM * m).flatten(1)).reshape(w.shape)
            ratio = w.shape[0] / math.prod(w.shape[1:])
            weights.append((1.0 - LR * DECAY) * w.double() - LR * max(1.0, ratio) ** 0.5 * o)
        return [*weights, *momenta]
    return _exact_loss(state)
