"""Orthogonalised updates of weights (the Muon optimiser), resident on the device.

The reference trains with Adam or its own Nadam (src/optimizer.py:6-113), which scale every weight by itself.  Here a weight is
a matrix - ``[out, in * kh * kw]`` of a dense or convolution layer - and its update the nearest (semi-)orthogonal matrix to its
momentum, so that all its directions learn at the same rate.  Not part of the reference's interface.
"""
import torch

from .layer import slayerCuda

#: The quintic whose slope at zero is as steep as it can be with every singular value ending near one.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_ADJUST = {None: 0, 'shape': 1, 'rms': 2}


def _coefficients(coefficients):
    a, b, c = (float(v) for v in coefficients)
    return a, b, c


def orthogonalize(matrix, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """A matrix ``[..., rows, cols]`` (float32, bfloat16 or float16; a stack of them in front) brought near the orthogonal factor
    of its polar decomposition by ``steps`` Newton-Schulz products: after ``X = matrix / (norm + eps)``, ``X`` becomes
    ``a X + (b A + c A A) X`` with ``A = X X^T`` (of a matrix with more rows than columns, its transpose's).

    With the default coefficients all singular values end between 0.68 and 1.13, those below 1/500 of the norm excepted.
    Matrices of all types are worked on with products of 22 bits (fewer where the norm is below a thousandth of ``eps`` and the result
    near zero: entries after the division are held to 2**-37).  No gradient flows through it.
    A matrix has at most 32768 rows or columns on its shorter side, 2**22 on the longer, and 2**31 elements."""
    if matrix.dim() < 2:
        raise ValueError("orthogonalize: a matrix has at least two dimensions, got %s" % (tuple(matrix.shape),))
    if matrix.requires_grad and torch.is_grad_enabled():
        raise ValueError("orthogonalize: no gradient flows through it; detach the matrix")
    return slayerCuda.orthogonalize(matrix.contiguous(), int(steps), *_coefficients(coefficients), float(eps))


@torch.no_grad()
def muonStep(weights, grads, momenta, lr, momentum=0.95, nesterov=True, weightDecay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
             adjust='shape'):
    """One optimiser step on lists of weights, in place, in one to three launches for up to 48 of them (fewer of the largest)::

        mom    = momentum * mom + grad
        update = orthogonalize(grad + momentum * mom if nesterov else mom)
        weight = weight * (1 - lr * weightDecay) - lr * factor * update

    A weight of shape ``[d0, d1, ...]`` is a matrix of ``d0`` rows.  Weights and their gradients are float32, bfloat16 or float16,
    momenta float32; none of them overlap, but for gradients.  ``factor`` is ``sqrt(max(1, rows / cols))`` (``adjust='shape'``),
    ``0.2 * sqrt(max(rows, cols))`` (``'rms'``: updates as large as Adam's) or 1 (``None``).  A call that is refused changes nothing.

    The products wait on barriers for a limited time.  If one ever runs out, weights may be partly updated, and
    ``capi.device_status()`` says 0x5103."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise ValueError("muonStep: %d weights, %d gradients, %d momenta" % (len(weights), len(grads), len(momenta)))
    if adjust not in _ADJUST:
        raise ValueError("muonStep: adjust must be one of %s, got %r" % (list(_ADJUST), adjust))
    seen = set()
    for w, g, m in zip(weights, grads, momenta):
        if w.dim() < 2:
            raise ValueError("muonStep: a weight has at least two dimensions, got %s" % (tuple(w.shape),))
        if g.is_sparse:
            raise ValueError("muonStep: sparse gradients are not taken")
        if not m.is_contiguous():
            raise ValueError("muonStep: momenta must be contiguous")
        if not w.is_contiguous() and any(n > 1 and s == 0 for n, s in zip(w.shape, w.stride())):
            raise ValueError("muonStep: a weight whose elements share memory")
        for t in (w, m):
            if t.numel() and t.data_ptr() in seen:
                raise ValueError("muonStep: the same weight or momentum twice")
            seen.add(t.data_ptr())
    if any(g.numel() and g.data_ptr() in seen for g in grads):
        raise ValueError("muonStep: a gradient in the memory of a weight or momentum")
    # a weight whose elements are in another order is updated in a copy
    there = [w if w.is_contiguous() else w.contiguous() for w in weights]
    slayerCuda.muonStep(there, [g.contiguous() for g in grads], momenta, float(lr), float(momentum), bool(nesterov), float(weightDecay),
                        _ADJUST[adjust], int(steps), *_coefficients(coefficients), float(eps))
    for w, t in zip(weights, there):
        if t is not w:
            w.copy_(t)


class Muon(torch.optim.Optimizer):
    """``muonStep`` as a PyTorch optimiser, for the weights of dense and convolution layers.  Parameters of fewer than two
    dimensions (delays, thresholds) belong to another optimiser.  The state of a parameter is its float32 ``'momentum'``, made by its
    first step: a step may be captured in a CUDA graph once every parameter has taken one (or a state was loaded)."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weightDecay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                 adjust='shape'):
        if not lr >= 0.0:
            raise ValueError("Muon: lr must not be negative, got %s" % lr)
        if not 0.0 <= momentum < 1.0:
            raise ValueError("Muon: momentum must lie in [0, 1), got %s" % momentum)
        if not weightDecay >= 0.0:
            raise ValueError("Muon: weightDecay must not be negative, got %s" % weightDecay)
        if adjust not in _ADJUST:
            raise ValueError("Muon: adjust must be one of %s, got %r" % (list(_ADJUST), adjust))
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weightDecay=weightDecay, steps=steps,
                                      coefficients=coefficients, eps=eps, adjust=adjust))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]['params']:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError("Muon: parameters have at least two dimensions, got %s" % (tuple(p.shape),))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts a state to its parameter's type: momenta keep their 32 bits
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        params = [p for group in self.param_groups for p in group['params']]
        for i, p in zip(ids, params):
            if 'momentum' in state_dict['state'].get(i, ()):
                self.state[p]['momentum'] = state_dict['state'][i]['momentum'].detach().to(p.device, torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        missing = [p for group in self.param_groups for p in group['params'] if p.grad is not None and 'momentum' not in self.state.get(p, ())]
        if any(p.is_cuda for p in missing) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("Muon: momenta that are made in a capture would be zero in every replay; take a step before the capture")
        for p in missing:
            self.state[p]['momentum'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        for group in self.param_groups:
            weights = [p for p in group['params'] if p.grad is not None]
            muonStep(weights, [p.grad for p in weights], [self.state[p]['momentum'] for p in weights],
                     **{k: group[k] for k in ('lr', 'momentum', 'nesterov', 'weightDecay', 'steps', 'coefficients', 'eps', 'adjust')})
        return loss
