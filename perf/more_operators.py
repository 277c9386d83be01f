"""What training over long sequences needs, as cases that can be timed and compared with their plain forms.

A psp filter forgets at one fixed rate, and a layer keeps float32 tensors of every time step for its backward pass.  Here are the leak
whose rate is an input, and the tensors kept in 8 bits:

``leak``       a gated leaky integrator over whole sequences, alone or with its gradient
``step``       one time step of it on a stream, its state updated in place
``restore``    a tensor compressed to 8 bits, and what it stands for then
``surrogate``  a membrane potential compressed, and the surrogate gradient of the spike function on it
``weight``     the input of a dense layer compressed, and the layer's weight gradient from it

Tensors are ``[N, C, 1, 1, T]``: N samples of C neurons, time last.
"""
import math

import torch

own = False

THETA, TAU, SCALE = 10.0, 10.0, 1.0     # surrogate gradient: SCALE / TAU * exp(-|u - THETA| / TAU)
GROUP = 32                              # time steps with one scale

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the hidden layer of the 2312-512-10 spiking classifier, batch 64: a gate for every neuron and step
        _leak("leak_mlp", 64, 512, 300, "float32", "full", "logit", True, False, False, True),
        # maps of a spiking CNN, 32 channels of 17 x 17: the largest work of all
        _leak("leak_cnn", 32, 9248, 300, "float32", "full", "logit", False, False, False, True),
        # a few long recordings: rows of an odd length, too few of them to fill the GPU
        _leak("leak_long", 2, 16, 65537, "bfloat16", "full", "decay", True, False, False, True),
        # learnable decays, one per neuron, over recordings of different lengths; the state goes in and comes out
        _leak("leak_neuron", 32, 256, 2000, "float32", "neuron", "logit", False, True, True, True),
        # a trained network on new data: no gradient
        _leak("leak_infer", 16, 1111, 145, "float16", "full", "logit", True, False, True, False),
        # one step of a stream: an experiment's network, bound by latency
        _step("step_mlp", 1, 512, "float32", "full", "logit", True),
        # one step of many streams
        _step("step_cnn", 64, 18496, "bfloat16", "neuron", "logit", False),
        # psp of the hidden layer kept for its backward pass
        _restore("restore_mlp", 64, 2312, 300, "float32"),
        # membrane potentials of 1450 steps, as the Loihi networks have
        _surrogate("surrogate_long", 64, 512, 1450),
        # an odd number of steps: rows that start anywhere
        _surrogate("surrogate_odd", 7, 1155, 301),
        # the 2312 -> 512 layer, batch 64
        _weight("weight_mlp", 64, 2312, 512, 300),
        # the 512 -> 10 layer behind it, an odd number of steps
        _weight("weight_out", 64, 512, 10, 301),
    ]


def _leak(name, N, C, T, dtype, gate, kind, coupled, state, ragged, train):
    return _named(name, {"op": "leak", "N": N, "C": C, "T": T, "dtype": dtype, "gate": gate, "kind": kind, "coupled": coupled, "state": state,
                         "ragged": ragged, "train": train})


def _step(name, N, C, dtype, gate, kind, coupled):
    return _named(name, {"op": "step", "N": N, "C": C, "dtype": dtype, "gate": gate, "kind": kind, "coupled": coupled})


def _restore(name, N, C, T, dtype):
    return _named(name, {"op": "restore", "N": N, "C": C, "T": T, "dtype": dtype})


def _surrogate(name, N, C, T):
    return _named(name, {"op": "surrogate", "N": N, "C": C, "T": T, "dtype": "float32"})


def _weight(name, N, C, O, T):
    return _named(name, {"op": "weight", "N": N, "C": C, "O": O, "T": T, "dtype": "float32"})


def _named(name, case):
    return {"name": name, **case} if name else case


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def yes():
        return rng.random() < 0.5

    op = rng.choice(["leak", "leak", "leak", "leak", "step", "restore", "surrogate", "weight", "weight"])
    dtype, gate = rng.choice(list(TYPES)), rng.choice(["full", "full", "neuron"])
    kind = rng.choice(["logit", "logit", "decay"])
    if op == "step":
        N = log(1, 64)
        return _step(None, N, max(1, log(1, 2000000) // N), dtype, gate, kind, yes())
    if op == "weight":
        N, T, C, O = log(1, 128), log(8, 2000), log(1, 8192), log(1, 1024)
        while 2.0 * N * T * C * O > 1.5e11 or N * T * (C + O) > 6e7:
            N, T = (N + 1) // 2, max(8, T * 2 // 3)
        return _weight(None, N, C, O, T)
    T = log(1, 100000) if op == "leak" and yes() else log(8, 2000)
    rows = max(1, log(max(64, T), 8e7) // T)
    N = min(rows, log(1, 64))
    C = rows // N
    if op == "leak":
        return _leak(None, N, C, T, dtype, gate, kind, yes(), yes(), yes(), rng.random() < 0.8)
    return _restore(None, N, C, T, dtype) if op == "restore" else _surrogate(None, N, C, T)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.empty(shape, device="cuda").normal_(generator=gen)


def _psp(gen, *shape):
    """Spikes of 5 % of the steps, filtered: what a layer's weights are applied to."""
    y = (torch.rand(shape, device="cuda", generator=gen) < 0.05).float()
    decay = 0.85
    for k in (1, 2, 4, 8):
        if k < shape[-1]:
            y[..., k:] += decay ** k * y[..., :-k].clone()
    return y


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = TYPES[case["dtype"]], case["op"]
    N, C, T = case["N"], case["C"], case.get("T", 1)
    state = {"case": dict(case)}
    if op in ("leak", "step"):
        shape = (N, C, 1, 1, T)
        gate = _normal(gen, *(shape if case["gate"] == "full" else (C, 1, 1, 1)))
        # from leaks of a few steps to some of a few hundred
        gate = gate.mul_(1.5).add_(2.5)
        if case["kind"] == "decay":
            gate = torch.sigmoid(gate)
        x = _normal(gen, *shape)
        if op == "step":
            state["x"], state["gate"] = x[..., 0].to(dtype), (gate[..., 0]).to(dtype)
            state["state"] = 2.0 * _normal(gen, N, C, 1, 1)
            return state
        state["x"], state["gate"] = x.to(dtype), gate.to(dtype)
        del x, gate
        state["initial"] = 2.0 * _normal(gen, N, C, 1, 1) if case["state"] else None
        state["lengths"] = None
        if case["ragged"]:      # more than half of the steps in most samples; one now and then is empty
            lengths = torch.randint(0, T + 1, (N,), device="cuda", generator=gen)
            lengths[: (N + 1) // 2] = torch.clamp(lengths[: (N + 1) // 2], min=(T + 1) // 2)
            state["lengths"] = lengths
        if case["train"]:
            state["upstream"] = _normal(gen, *shape).to(dtype)
            state["upstream_state"] = _normal(gen, N, C, 1, 1)
            for k in ("x", "gate", "initial"):
                if state[k] is not None:
                    state[k].requires_grad_(True)
        return state
    if op == "surrogate":
        state["x"] = 6.0 * _normal(gen, N, C, 1, 1, T)
        state["upstream"] = _normal(gen, N, C, 1, 1, T)
        return state
    state["x"] = _psp(gen, N, C, 1, 1, T).to(dtype)
    if op == "weight":
        state["upstream"] = _normal(gen, N, case["O"], 1, 1, T)
    return state


# ---------------------------------------------------------------------------------------- the plain forms
def _scan(r, y):
    """y_t + f_t y_{t-1} + f_t f_{t-1} y_{t-2} ... along the last dimension, by doubling, with f = 1 - r.  Slow leaks are next to one, where
    32 bits hold r better than f: what a rounding of f takes from every step adds up over a state's memory."""
    r, y = r.clone(), y.clone()
    k, T = 1, y.shape[-1]
    while k < T:
        y[..., k:] += y[..., :-k] - r[..., k:] * y[..., :-k]
        r[..., k:] = r[..., k:] + (r[..., :-k] - r[..., k:] * r[..., :-k])
        k *= 2
    return y


def _decay(gate, kind):
    """(f, 1 - f) in 32 bits."""
    gate = gate.float()
    return (1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))) if kind == "logit" else (gate, 1.0 - gate)


def _plain_leak(state):
    case = state["case"]
    x, gate = state["x"].detach(), state["gate"].detach()
    shape, T = x.shape, x.shape[-1]
    f, rest = _decay(gate, case["kind"])
    u = x.float() * rest if case["coupled"] else x.float()
    r = rest.expand(shape)
    there = None
    if state["lengths"] is not None:
        there = torch.arange(T, device=x.device) < state["lengths"][:, None, None, None, None]
        r, u = torch.where(there, r, 0.0), torch.where(there, u, 0.0)       # the state stays what it is
    first = torch.zeros(shape[:-1], device=x.device) if state["initial"] is None else state["initial"].detach()
    u = u.clone()
    u[..., 0] += first - r[..., 0] * first
    y = _scan(r, u)
    out = (y if there is None else torch.where(there, y, 0.0)).to(x.dtype)
    outs = [out, y[..., -1]] if case["state"] else [out]
    if not case["train"]:
        return outs
    g = state["upstream"].float()
    if there is not None:
        g = torch.where(there, g, 0.0)
    if case["state"]:
        g = g.clone()
        g[..., -1] += state["upstream_state"]
    after = torch.cat([torch.zeros_like(r[..., :1]), r[..., 1:].flip(-1)], -1)
    lam = _scan(after, g.flip(-1)).flip(-1)
    before = torch.cat([first[..., None], y[..., :-1]], -1)
    dx = lam * rest if case["coupled"] else lam
    df = lam * (before - x.float()) if case["coupled"] else lam * before
    first_grad = lam[..., 0] - r[..., 0] * lam[..., 0]
    if there is not None:
        dx, df = torch.where(there, dx, 0.0), torch.where(there, df, 0.0)
    if case["gate"] != "full":
        df = df.double().sum((0, 2, 3, 4)).reshape(gate.shape)
    dgate = df * (f * rest) if case["kind"] == "logit" else df
    outs += [dx.to(x.dtype), dgate.to(gate.dtype)]
    return outs + [first_grad] if case["state"] else outs


def _plain_step(state):
    case = state["case"]
    f, rest = _decay(state["gate"], case["kind"])
    u = state["x"].float() * rest if case["coupled"] else state["x"].float()
    state["state"].mul_(f).add_(u)
    return state["state"].to(state["x"].dtype)


def _plain_compress(x):
    """What 8 bits hold of x: whole multiples, up to 127, of a power of two for every GROUP steps of a row."""
    T = x.shape[-1]
    x = torch.nn.functional.pad(x.detach().float(), (0, -T % GROUP)).unflatten(-1, (-1, GROUP))
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    # the smallest power with amax <= 127 * 2**power, within what a float can be
    scale = torch.exp2(torch.clamp(exponent - 7 + (mantissa > 127.0 / 128.0), -126, 121).double()).float()
    return (torch.clamp(torch.round(x / scale), -127, 127) * scale).flatten(-2)[..., :T]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case, op = state["case"], state["case"]["op"]
    if op == "leak":
        if not own:
            return _plain_leak(state)
        from slayerpytorch_b200.recurrence import gatedLeak
        with torch.set_grad_enabled(case["train"]):
            y = gatedLeak(state["x"], state["gate"], initial=state["initial"], lengths=state["lengths"], kind=case["kind"],
                          coupled=case["coupled"], returnState=case["state"])
        outs = list(y) if case["state"] else [y]
        if not case["train"]:
            return outs
        leaves = [state["x"], state["gate"]] + ([state["initial"]] if case["state"] else [])
        grads = torch.autograd.grad(outs, leaves, [state["upstream"], state["upstream_state"]][: len(outs)])
        return [*(o.detach() for o in outs), *grads]
    if op == "step":
        if own:
            from slayerpytorch_b200.recurrence import gatedLeakStep
            return [gatedLeakStep(state["x"], state["gate"], state["state"], kind=case["kind"], coupled=case["coupled"]), state["state"]]
        return [_plain_step(state), state["state"]]
    if own:
        from slayerpytorch_b200 import checkpoint
        kept = checkpoint.compress(state["x"])
        if op == "restore":
            return kept.restore()
        if op == "surrogate":
            return checkpoint.spikeGrad(state["upstream"], kept, THETA, TAU, SCALE)
        return checkpoint.weightGrad(state["upstream"], kept)
    kept = _plain_compress(state["x"])
    if op == "restore":
        return kept.to(state["x"].dtype)
    if op == "surrogate":
        return state["upstream"] * (SCALE / TAU * torch.exp(-(kept - THETA).abs() / TAU))
    N, C, O, T = (case[k] for k in "NCOT")
    g = state["upstream"].reshape(N, O, T).transpose(0, 1).reshape(O, N * T)
    return (g @ kept.reshape(N, C, T).transpose(0, 1).reshape(C, N * T).T).reshape(O, C, 1, 1, 1)


def work(case):
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    op, rows = case["op"], case["N"] * case["C"]
    gates = rows if case.get("gate") == "full" else case["C"]
    if op == "step":
        return {"bytes": 2 * size * rows + size * gates + 8 * rows, "flops": 6 * rows}
    T = case["T"]
    if op == "leak":
        if case["gate"] == "full":
            gates *= T
        states = 4 * rows if case["state"] else 0
        if case["train"]:       # x, gate and the upstream gradient; outputs, and the gradients of x and the gate
            return {"bytes": size * (4 * rows * T + 2 * gates) + 4 * states, "flops": 16 * rows * T}
        return {"bytes": size * (2 * rows * T + gates) + 2 * states, "flops": 6 * rows * T}
    if op == "restore":
        return {"bytes": 2 * size * rows * T, "flops": 4 * rows * T}
    if op == "surrogate":
        return {"bytes": 12 * rows * T, "flops": 10 * rows * T}
    N, C, O = case["N"], case["C"], case["O"]
    return {"bytes": 4 * (N * T * (C + O) + O * C), "flops": 2 * N * T * C * O}


# ---------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_leak(state):
    """A step after another, in double."""
    case = state["case"]
    shape, T, N = state["x"].shape, case["T"], case["N"]
    rows = shape[0] * shape[1]
    steps = lambda v: v.detach().expand(shape).reshape(rows, T).t().contiguous()  # noqa: E731
    x, gate = steps(state["x"]), steps(state["gate"])
    lengths = torch.full((N,), T, device=x.device) if state["lengths"] is None else state["lengths"]
    lengths = lengths.repeat_interleave(case["C"])
    logit = case["kind"] == "logit"

    def leak(t):
        return torch.sigmoid(gate[t].double()) if logit else gate[t].double()

    h = torch.zeros(rows, dtype=torch.float64, device=x.device) if state["initial"] is None else state["initial"].detach().double().reshape(rows)
    before = torch.empty((T, rows), dtype=torch.float64, device=x.device) if case["train"] else None
    y = torch.empty((T, rows), dtype=torch.float64, device=x.device)
    for t in range(T):
        f, v, on = leak(t), x[t].double(), t < lengths
        if before is not None:
            before[t] = h
        h = torch.where(on, f * h + ((1.0 - f) * v if case["coupled"] else v), h)
        y[t] = h * on
    back = lambda v: v.t().reshape(shape)  # noqa: E731
    outs = [back(y), h.reshape(shape[:-1])] if case["state"] else [back(y)]
    if not case["train"]:
        return outs
    del y
    g = steps(state["upstream"])
    lam = state["upstream_state"].double().reshape(rows).clone() if case["state"] else torch.zeros(rows, dtype=torch.float64, device=x.device)
    dx = torch.empty_like(before)
    for t in range(T - 1, -1, -1):
        f, v, on = leak(t), x[t].double(), t < lengths
        lam = torch.where(on, lam + g[t].double(), lam)
        slope = lam * (before[t] - v if case["coupled"] else before[t]) * on
        dx[t] = lam * on * ((1.0 - f) if case["coupled"] else 1.0)
        before[t] = slope * f * (1.0 - f) if logit else slope       # the gate's gradient takes the state's place
        lam = torch.where(on, lam * f, lam)
    dgate = back(before)
    if case["gate"] != "full":
        dgate = dgate.sum((0, 4))[..., None]
    outs += [back(dx), dgate]
    return outs + [lam.reshape(shape[:-1])] if case["state"] else outs


def _exact_compress(x):
    x = x.detach().double()
    parts = []
    for part in x.split(GROUP, -1):
        top = part.abs().amax(-1, keepdim=True) / 127.0
        power = torch.where(top > 0, torch.log2(top.clamp(min=1e-300)).ceil(), torch.zeros_like(top))
        # what the logarithm rounded away
        power = torch.where((top > 0) & (top <= 2.0 ** (power - 1.0)), power - 1.0, power)
        power = torch.where(top > 2.0 ** power, power + 1.0, power).clamp(-126.0, 121.0)
        parts.append((part / 2.0 ** power).round().clamp(-127, 127) * 2.0 ** power)
    return torch.cat(parts, -1)


def exact(case, seed):
    if case["op"] == "leak" and case["T"] * (2 if case["train"] else 1) > 150000:
        return None
    state = prepare(case, seed)
    if case["op"] == "leak":
        return _exact_leak(state)
    if case["op"] == "step":
        f = state["gate"].double()
        f = torch.sigmoid(f) if case["kind"] == "logit" else f
        h = f * state["state"].double() + state["x"].double() * ((1.0 - f) if case["coupled"] else 1.0)
        return [h, h]
    kept = _exact_compress(state["x"])
    if case["op"] == "restore":
        return kept
    if case["op"] == "surrogate":
        return state["upstream"].double() * SCALE / TAU * torch.exp((kept - THETA).abs() / -TAU)
    grad = torch.zeros((case["O"], case["C"]), dtype=torch.float64, device="cuda")
    for n in range(case["N"]):
        grad.addmm_(state["upstream"][n].double().flatten(0, 2), kept[n].flatten(0, 2).T)
    return grad.reshape(case["O"], case["C"], 1, 1, 1)
