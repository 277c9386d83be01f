"""The gated leaky integrator: a psp filter whose decay is an input.

``psp`` (src/slayer.py:125-140 of the reference) forgets at one fixed rate.  Here every neuron, or every neuron and time step, has a
decay of its own, which is learned or computed by the network, so that a layer can hold something over thousands of steps and
drop it in one.  Tensors are ``[..., T]`` as everywhere, time last.  Not part of the reference's interface.
"""
import torch

from . import load_ops

slayerCuda, _ = load_ops()

_KINDS = {'logit': 1, 'decay': 0}


def _flags(op, kind, coupled):
    if kind not in _KINDS:
        raise ValueError("%s: kind must be one of %s, got %r" % (op, sorted(_KINDS), kind))
    return _KINDS[kind] + (2 if coupled else 0)


def gatedLeak(x, gate, initial=None, lengths=None, kind='logit', coupled=False, returnState=False):
    """A leaky integrator over whole sequences, or over the next part of a stream::

        y_t = f_t * y_{t-1} + x_t                   (coupled: f_t * y_{t-1} + (1 - f_t) * x_t)

    with ``f = sigmoid(gate)`` (``kind='logit'``) or ``f = gate`` (``'decay'``: from 0 to 1; values outside are taken as they are, with less
    exact results where -1 is near, and products that may overflow where single steps do not).  ``x [..., T]``: float32, bfloat16 or float16, any strides (a copy is made where it is not
    contiguous); ``y`` is like it.  ``gate`` broadcasts to ``x``: one of the shape of ``x`` (or with a time dimension of ``T``) has
    the type of ``x``; one per neuron, ``[C, H, W, 1]`` say, may have any of the three, and is not copied where its dimensions lie
    next to each other.  ``initial [...]``: the state before the first step (default 0).

    ``lengths`` holds a number of steps for each of ``x.shape[0]`` samples (int64 or int32, taken into [0, T]): the steps behind it are not
    used, whatever they hold, ``y`` and all gradients are 0 there, and the state stays what it was.  With ``returnState`` the
    state after the last step comes too, float32, of the shape of ``initial``.

    Differentiable once in ``x``, ``gate`` and ``initial``.  Results are off by a few steps of float32, however slow the leak.  Nothing but
    ``x``, ``gate`` and one float32 state for 12 or 16 steps is kept for the backward pass.  A state that is not finite makes those after it so, as NaN
    possibly where the formula gives an infinity (here and in ``gatedLeakStep``)."""
    out = slayerCuda.gatedLeak(x, gate, initial, lengths, _flags("gatedLeak", kind, coupled), returnState)
    return (out[0], out[1]) if returnState else out[0]


def gatedLeakStep(x, gate, state, kind='logit', coupled=False):
    """One time step of ``gatedLeak`` on a stream, in one launch: ``x [...]``, ``gate`` broadcasting to it (any of the three types), ``state``
    of the shape of ``x``, float32 and contiguous, updated in place; it may not share memory with the other two.  Returns the new
    state in the type of ``x``.  No gradient flows through it."""
    return slayerCuda.gatedLeakStep(x, gate, state, _flags("gatedLeakStep", kind, coupled))
