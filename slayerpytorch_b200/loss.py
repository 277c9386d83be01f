"""Spike losses, losses of choices, and the spike-count classifier, resident on the device.

Same names, arguments and results as ``spikeLoss`` (src/spikeLoss.py:7-104) and
``spikeClassifier`` (src/spikeClassifier.py:4-22) of the reference, which the layers of the
hot path feed in every training step.  The reference computes the spike counts, the desired
counts and the target-region mask with NumPy on the host, which costs a device-to-host copy of
the full output spike tensor, a host-to-device copy of two tensors of the same size and two
synchronisations per step (src/spikeLoss.py:91-102).  Here every term is a tensor expression
on the device of ``spikeOut``; nothing is copied and nothing waits.

Arithmetic follows the reference closely enough for identical results: the spike-count error
is formed in float64 (NumPy promotes ``float32 - int64`` to float64 there) and rounded to
float32 once, and the part of the output inside the target region is treated as a constant
in the backward pass, exactly as the reference's ``spikeDesired`` built from ``.data`` is.

Where there is no desired answer but a judgement of the one given, ``policyLoss`` and ``preferenceLoss`` take rows of logits and
the entry chosen in each (``actionLogProb`` gives the values of the policy that chose); ``spikeLoss.policy`` and
``spikeLoss.preference`` take the logits from the output neurons' spike counts.  They have first derivatives only.
"""
import numpy as np
import torch

from .layer import slayerCuda, spikeLayer


class _NumSpikesFunction(torch.autograd.Function):
    """Value and gradient of the spike-count loss from one kernel (``slayerCuda.numSpikesLoss``):
    forward keeps the gradient for a unit upstream gradient, backward scales it."""

    @staticmethod
    def forward(ctx, spikeOut, desiredCount, srmKernel, start, stop, Ts, scale):
        sq, grad = slayerCuda.numSpikesLoss(spikeOut.contiguous(), desiredCount, srmKernel, start, stop, Ts, scale)
        ctx.save_for_backward(grad)
        return (sq * (0.5 * Ts)).float()

    @staticmethod
    def backward(ctx, gradLoss):
        (grad,) = ctx.saved_tensors
        return grad * gradLoss, None, None, None, None, None, None


# ------------------------------------------------------------------- choices: rows of logits, one entry each
def actionLogProb(logits, action, mask=None, scale=1.0):
    """Log-probability of one chosen entry of each row: ``log softmax(scale * logits)[action]``, float32, of the shape of
    ``action``; 0 where ``mask`` is false (those rows are not read), NaN where the action lies outside.

    ``logits [..., V]``: float32, bfloat16 or float16, any strides (rows whose entries are apart are copied).  Differentiable in
    ``logits``.  It is what ``policyLoss`` and ``preferenceLoss`` take as old and reference values.  Not part of the
    reference's interface."""
    return slayerCuda.actionLogProb(logits, action, mask, float(scale))


def policyLoss(logits, action, oldLogProb, advantage, refLogProb=None, mask=None, clip=0.2, klCoef=0.0, scale=1.0, reduction='sum',
               returnLogProb=False):
    """Clipped policy loss of the choices a network made, with an optional KL term that holds it to a reference.

    ``logits [..., V]`` (float32, bfloat16, float16); ``action``, ``oldLogProb``, ``refLogProb`` and ``mask`` have its shape without
    ``V``; ``advantage`` too, or without the last dimension of that as well (one per sequence).  Per row, with ``lp`` the chosen
    entry's log-probability under ``softmax(scale * logits)``::

        ratio = exp(lp - oldLogProb)
        loss  = -min(ratio * advantage, clip(ratio, 1 - low, 1 + high) * advantage)
                + klCoef * (exp(refLogProb - lp) - (refLogProb - lp) - 1)

    ``clip`` is ``(low, high)`` or one number for both.  ``reduction``: ``'sum'`` (as the spike losses add up their batch, so that
    gradients of shards add), ``'mean'`` over the rows that ``mask`` keeps, or ``'sequence'``: the mean over the sequences (all
    dimensions but the last of ``action``) of the mean over each one's kept rows; over no rows a mean is 0.  Masked rows are not
    read and have gradient 0.  Old and reference values and advantages are constants.

    The value and the gradient come from one pass; the gradient is formed again where the loss is multiplied by something before
    ``backward()``, so a constant factor is cheaper in ``advantage`` and ``klCoef``.  With ``returnLogProb`` the rows'
    log-probabilities come too (no gradient).  Not part of the reference's interface."""
    kinds = {'sum': 0, 'mean': 1, 'sequence': 2}
    if reduction not in kinds:
        raise ValueError("policyLoss: reduction must be one of %s, got %r" % (sorted(kinds), reduction))
    low, high = (float(c) for c in (clip if isinstance(clip, (tuple, list)) else (clip, clip)))
    if not (low >= 0.0 and high >= 0.0):
        raise ValueError("policyLoss: the clip range must not be negative, got %s" % (clip,))
    if (klCoef != 0.0) != (refLogProb is not None):
        raise ValueError("policyLoss: klCoef and refLogProb belong together")
    loss, logp = slayerCuda.policyLoss(logits, action, oldLogProb, advantage, refLogProb, mask, low, high, float(klCoef), float(scale),
                                       kinds[reduction])
    return (loss, logp) if returnLogProb else loss


def preferenceLoss(logits, action, refLogProb, pairs=None, mask=None, beta=0.1, labelSmoothing=0.0, scale=1.0, reduction='sum'):
    """Loss of paired sequences of choices, of which the first is preferred to the second.

    ``logits [S, L, V]`` (float32, bfloat16, float16), ``action`` and ``mask`` ``[S, L]``; ``refLogProb [S]``: each sequence's summed
    log-probability under the reference; ``pairs`` ``[P, 2]`` int64 sequence indices, the preferred one first (default: sequence
    ``i`` against ``i + S / 2``); a sequence may be in several pairs.  With ``m`` a sequence's summed log-probability of its choices
    (those that ``mask`` keeps) minus ``refLogProb``, and ``h = beta * (m[first] - m[second])``::

        loss = -(1 - labelSmoothing) * log sigmoid(h) - labelSmoothing * log sigmoid(-h)

    summed over the pairs (``'sum'``) or their mean.  Not part of the reference's interface."""
    kinds = {'sum': 0, 'mean': 1}
    if reduction not in kinds:
        raise ValueError("preferenceLoss: reduction must be one of %s, got %r" % (sorted(kinds), reduction))
    if not 0.0 <= labelSmoothing <= 1.0:
        raise ValueError("preferenceLoss: labelSmoothing must lie between 0 and 1, got %s" % labelSmoothing)
    return slayerCuda.preferenceLoss(logits, action, refLogProb, pairs, mask, float(beta), float(labelSmoothing), float(scale), kinds[reduction])


class spikeLoss(torch.nn.Module):
    """``spikeLoss(networkDescriptor, slayerClass=spikeLayer)`` with ``networkDescriptor`` holding
    ``'neuron'``, ``'simulation'`` and ``'training': {'error': ...}`` (src/spikeLoss.py:30-37)."""

    def __init__(self, networkDescriptor, slayerClass=spikeLayer):
        super().__init__()
        self.neuron = networkDescriptor['neuron']
        self.simulation = networkDescriptor['simulation']
        self.errorDescriptor = networkDescriptor['training']['error']
        self.slayer = slayerClass(self.neuron, self.simulation)
        self.fused = True          # numSpikes: one fused kernel; False = the tensor expressions

    def spikeTime(self, spikeOut, spikeDesired):
        """Van Rossum-like distance between two spike trains (src/spikeLoss.py:39-59)."""
        assert self.errorDescriptor['type'] == 'SpikeTime', "Error type is not SpikeTime"
        error = self.slayer.psp(spikeOut - spikeDesired)
        return 1 / 2 * torch.sum(error ** 2) * self.simulation['Ts']

    def numSpikes(self, spikeOut, desiredClass, numSpikesScale=1):
        """Spike-count loss inside the target region, spike-time loss outside of it
        (src/spikeLoss.py:61-104).  ``desiredClass`` is one-hot with a time dimension of 1."""
        assert self.errorDescriptor['type'] == 'NumSpikes', "Error type is not NumSpikes"
        region = self.errorDescriptor['tgtSpikeRegion']
        count = self.errorDescriptor['tgtSpikeCount']
        Ts = self.simulation['Ts']
        start = int(np.rint(region['start'] / Ts))
        stop = int(np.rint(region['stop'] / Ts))
        T = spikeOut.shape[-1]
        lo, hi = slice(start, stop).indices(T)[:2]        # the slice the reference takes, made explicit

        if spikeOut.is_cuda and spikeOut.dtype == torch.float32 and self.fused and stop != start and T <= 8192:
            # one kernel for the loss and its gradient (same arithmetic as the expressions below); rows of up to
            # 8192 steps fit its shared memory with any filter (2 words per step, and 3 per tap, of which T count)
            onehot = desiredClass.to(spikeOut.device)
            desired = torch.where(onehot == True, float(count[True]), float(count[False]))    # noqa: E712
            desired = desired.to(torch.float32).expand(spikeOut.shape[:-1] + (1,)).reshape(-1).contiguous()
            return _NumSpikesFunction.apply(spikeOut, desired, self.slayer.srmKernel, start, stop, float(Ts),
                                            float(numSpikesScale))

        with torch.no_grad():
            inside = torch.zeros(T, dtype=spikeOut.dtype, device=spikeOut.device)
            inside[lo:hi] = 1
            actual = torch.sum(spikeOut[..., start:stop], 4, keepdim=True) * Ts          # float32, as the reference
            desired = torch.where(desiredClass.to(spikeOut.device) == True,              # noqa: E712 (tensor compare)
                                  torch.tensor(float(count[True]), dtype=torch.float64, device=spikeOut.device),
                                  torch.tensor(float(count[False]), dtype=torch.float64, device=spikeOut.device))
            count_error = (actual.double() - desired) / (stop - start) * numSpikesScale  # float64
            count_term = (count_error * inside.double()).float()                         # rounded once
            spikeDesired = inside * spikeOut                                             # constant in backward

        error = self.slayer.psp(spikeOut - spikeDesired)
        error = error + count_term
        return 1 / 2 * torch.sum(error ** 2) * Ts

    def _countLogits(self, spikeOut):
        """Spike counts inside the target region, one row per sample: what the network's choice is drawn from."""
        region = self.errorDescriptor['tgtSpikeRegion']
        Ts = self.simulation['Ts']
        start, stop = int(np.rint(region['start'] / Ts)), int(np.rint(region['stop'] / Ts))
        return torch.sum(spikeOut[..., start:stop], -1).reshape(spikeOut.shape[0], spikeOut.shape[1:-1].numel()) * Ts

    def actionLogProb(self, spikeOut, action):
        """Log-probability of each sample's choice among the output neurons: a softmax of ``countScale`` times their spike counts
        inside the target region.  Takes error types ``'Policy'`` and ``'Preference'``; not part of the reference's interface."""
        assert self.errorDescriptor['type'] in ('Policy', 'Preference'), "Error type is neither Policy nor Preference"
        counts = self._countLogits(spikeOut)
        return actionLogProb(counts, action.reshape(-1), scale=self.errorDescriptor.get('countScale', 1.0)).reshape(action.shape)

    def policy(self, spikeOut, action, oldLogProb, advantage, refLogProb=None, mask=None):
        """``policyLoss`` of choices drawn from the output neurons' spike counts, one per sample, summed over the batch.
        The error descriptor: ``{'type': 'Policy', 'tgtSpikeRegion': {'start', 'stop'}, 'countScale': 1.0, 'clip': 0.2, 'klCoef': 0.0}``
        (the last three may be missing).  Not part of the reference's interface."""
        assert self.errorDescriptor['type'] == 'Policy', "Error type is not Policy"
        e = self.errorDescriptor
        return policyLoss(self._countLogits(spikeOut), action, oldLogProb, advantage, refLogProb=refLogProb, mask=mask,
                          clip=e.get('clip', 0.2), klCoef=e.get('klCoef', 0.0), scale=e.get('countScale', 1.0))

    def preference(self, spikeOut, action, refLogProb, pairs=None, mask=None):
        """``preferenceLoss`` of episodes of choices: ``action [S, L]``, and ``spikeOut`` holds the S * L samples in that order; summed
        over the pairs.  The error descriptor: ``{'type': 'Preference', 'tgtSpikeRegion': {'start', 'stop'}, 'countScale': 1.0,
        'beta': 0.1, 'labelSmoothing': 0.0}`` (the last three may be missing).  Not part of the reference's interface."""
        assert self.errorDescriptor['type'] == 'Preference', "Error type is not Preference"
        e = self.errorDescriptor
        counts = self._countLogits(spikeOut)
        if action.dim() != 2 or action.numel() != counts.shape[0]:
            raise ValueError("preference: action must be [sequences, choices] with one entry per sample, got %s for %d samples"
                             % (tuple(action.shape), counts.shape[0]))
        return preferenceLoss(counts.reshape(action.shape + counts.shape[1:]), action, refLogProb, pairs=pairs, mask=mask, beta=e.get('beta', 0.1),
                              labelSmoothing=e.get('labelSmoothing', 0.0), scale=e.get('countScale', 1.0))


class spikeClassifier:
    """Class label = the output neuron with the most spikes (src/spikeClassifier.py:9-20).

    As in the reference the labels come back as a CPU tensor, so that the reference's training
    scripts, which compare them with the CPU labels of a DataLoader
    (``torch.sum(getClass(output) == label)``), run unchanged; the counting itself stays on the
    device and only one index per sample crosses.  ``host=False`` keeps the result on the device
    of ``spike`` (no synchronisation)."""

    @staticmethod
    def getClass(spike, host=True):
        numSpikes = torch.sum(spike, 4, keepdim=True)
        labels = torch.max(numSpikes.reshape((numSpikes.shape[0], -1)), 1)[1]
        return labels.cpu() if host else labels
