"""Tensors of a layer kept in 8 bits until its backward pass.

Backpropagation through time needs every layer's input and membrane potential of every time step again (``ctx.save_for_backward`` in
src/slayer.py:824-866 of the reference), and over long sequences that is what fills the memory.  ``compress`` keeps such a tensor in
33/128 of float32's bytes, and the two uses that a layer has for it read it as it is: the surrogate gradient of the spike
function, and the weight gradient of a dense layer.  ``spikeLayer.spike(u, checkpoint=True)`` and
``spikeLayer.dense(..., checkpoint=True)`` do all of it.  The forward pass is not changed by any of this; gradients are those of
inputs that are off by at most 1/127 of the largest of their 32 steps.  Not part of the reference's interface.
"""
import torch

from . import load_ops

slayerCuda, _ = load_ops()


class Checkpoint:
    """A tensor ``[..., T]`` in 8 bits, made by ``compress``: ``q`` (int8, ``[rows, 32 * groups]``) and ``scale`` (uint8,
    ``[groups, rows]``, one for each 32 steps of a row: the values are ``q * 2**(scale - 127)``)."""

    def __init__(self, q, scale, shape, dtype):
        self.q, self.scale, self.shape, self.dtype = q, scale, torch.Size(shape), dtype

    def restore(self, dtype=None):
        """What the 8 bits stand for, in the type that was compressed, or another (rounded to it).  In float16 65536 is 65504, the type's largest
        number: what is finite there comes back finite."""
        dtype = self.dtype if dtype is None else dtype
        return slayerCuda.restore8(self.q, self.scale, self.shape, torch.empty((), dtype=dtype))


def compress(x):
    """``x [..., T]`` (float32, bfloat16 or float16; a copy is made where it is not contiguous) in 8 bits: of each 32 consecutive steps of a
    row, whole multiples up to 127 of the smallest power of two (from 2**-126 to 2**121) that allows it, rounded to nearest, ties to
    even.  Values that are not finite come back as NaN and do not change the others.  Rows are held in whole groups: a row of fewer
    than 32 steps takes 33 bytes.  No gradient flows through it."""
    q, scale = slayerCuda.compress8(x)
    return Checkpoint(q, scale, x.shape, x.dtype)


def spikeGrad(grad, kept, theta, tau, scale):
    """``grad * (scale / tau * exp(-|u - theta| / tau))`` with ``u`` what ``kept`` stands for: the surrogate gradient of the spike function
    (src/slayer.py:858-865), float32, on a membrane potential kept by ``compress``."""
    if grad.shape != kept.shape:
        raise ValueError("spikeGrad: grad must have the shape of what was compressed, %s, got %s" % (tuple(kept.shape), tuple(grad.shape)))
    return slayerCuda.spikeGrad8(grad.contiguous(), kept.q, kept.scale, float(theta), float(tau), float(scale))


def weightGrad(grad, kept):
    """Weight gradient of a dense layer: ``grad [N, O, 1, 1, T]`` (float32) of its output, ``kept`` its input ``[N, C, H, W, T]`` kept by
    ``compress``; returns ``[O, C, H, W, 1]``, the sum over samples and steps of ``grad * input``, to float32 precision and the same
    in every call.  Any number of dimensions from three on.  Of gradients below 2**-110 what lies under 2**-133 has no part in it; where one is not
    finite, or an input was not, the sums that it is in are NaN."""
    return slayerCuda.weightGrad8(grad.contiguous(), kept.q, kept.scale, kept.shape)
