"""CPU: what the losses of choices refuse, and what their C entries do before they touch a GPU."""
import ctypes

import pytest
import torch

from slayerpytorch_b200 import capi, loss


def test_shapes_types_and_options_are_checked():
    x, a, z = torch.zeros(4, 3, 6), torch.zeros(4, 3, dtype=torch.long), torch.zeros(4, 3)
    with pytest.raises(ValueError, match="action must have the shape"):
        loss.actionLogProb(x, a[:, :2])
    with pytest.raises(TypeError, match="int64 or int32"):
        loss.actionLogProb(x, z)
    with pytest.raises(ValueError, match="mask must have the shape"):
        loss.actionLogProb(x, a, mask=z[:1])
    with pytest.raises(ValueError, match="at least one entry"):
        loss.actionLogProb(x[..., :0], a)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            loss.actionLogProb(x, a, scale=scale)
    with pytest.raises(ValueError, match="reduction"):
        loss.policyLoss(x, a, z, z, reduction="none")
    with pytest.raises(ValueError, match="clip"):
        loss.policyLoss(x, a, z, z, clip=(0.2, -0.1))
    with pytest.raises(ValueError, match="clip"):
        loss.policyLoss(x, a, z, z, clip=float("nan"))
    with pytest.raises(ValueError, match="belong together"):
        loss.policyLoss(x, a, z, z, klCoef=0.1)
    with pytest.raises(ValueError, match="belong together"):
        loss.policyLoss(x, a, z, z, refLogProb=z)
    with pytest.raises(ValueError, match="oldLogProb"):
        loss.policyLoss(x, a, z[:, :1], z)
    with pytest.raises(ValueError, match="advantage"):
        loss.policyLoss(x, a, z, z[:1])
    with pytest.raises(ValueError, match="needs a dimension"):
        loss.policyLoss(x[0, 0], a[0, 0], z[0, 0], z[0, 0], reduction="sequence")
    with pytest.raises(ValueError, match="sequences, choices, entries"):
        loss.preferenceLoss(x[0], a[0], z[:, 0])
    with pytest.raises(ValueError, match="refLogProb"):
        loss.preferenceLoss(x, a, z)
    with pytest.raises(ValueError, match="even"):
        loss.preferenceLoss(x[:3], a[:3], z[:3, 0])
    with pytest.raises(ValueError, match="pairs"):
        loss.preferenceLoss(x, a, z[:, 0], pairs=a)
    with pytest.raises(ValueError, match="labelSmoothing"):
        loss.preferenceLoss(x, a, z[:, 0], labelSmoothing=1.5)
    with pytest.raises(ValueError, match="reduction"):
        loss.preferenceLoss(x, a, z[:, 0], reduction="sequence")


def test_cpu_tensors_are_refused():
    x, a, z = torch.zeros(4, 3, 6), torch.zeros(4, 3, dtype=torch.long), torch.zeros(4, 3)
    for call in (lambda: loss.actionLogProb(x, a), lambda: loss.policyLoss(x, a, z, z), lambda: loss.preferenceLoss(x, a, z[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_error_types_of_the_spike_losses():
    d = {"neuron": {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1},
         "simulation": {"Ts": 1.0, "tSample": 20}, "training": {"error": {"type": "SpikeTime", "tgtSpikeRegion": {"start": 0, "stop": 20}}}}
    net = loss.spikeLoss(d)
    s, a, z = torch.zeros(4, 3, 1, 1, 20), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    for call in (lambda: net.policy(s, a, z, z), lambda: net.preference(s, a.reshape(2, 2), z[:2]), lambda: net.actionLogProb(s, a)):
        with pytest.raises(AssertionError):
            call()
    d["training"]["error"]["type"] = "Preference"
    with pytest.raises(ValueError, match="one entry per sample"):
        net.preference(s, a[:3, None], z[:3])


def test_c_entries_check_their_arguments():
    lib = capi.load()
    null, p, q = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(32)
    lp = lambda **k: lib.slayer_b200_log_prob(*{**dict(  # noqa: E731
        logp=p, stats=null, logits=q, dtype=0, action=p, mask=null, rows=2, V=5, stride=5, scale=1.0, stream=null), **k}.values())
    for bad in (dict(rows=-1), dict(V=0), dict(stride=-1), dict(dtype=3), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(logits=null), dict(action=null), dict(logp=null)):
        assert lp(**bad) == -1, bad
        assert lib.slayer_b200_last_error()
    assert lp(V=1 << 31) == -3
    assert lp(rows=0, logits=null) == 0
    pl = lambda **k: lib.slayer_b200_policy_loss(*{**dict(  # noqa: E731
        loss=p, grad=null, logp=null, stats=p, coef=p, workspace=p, logits=q, dtype=0, action=p, old=p, adv=p, adv_len=1, ref=null, mask=null,
        rows=6, seq_len=3, V=5, stride=5, scale=1.0, lo=0.2, hi=0.2, kl=0.0, reduction=0, stream=null), **k}.values())
    for bad in (dict(loss=null), dict(lo=-0.1), dict(hi=float("nan")), dict(reduction=3), dict(adv_len=0), dict(seq_len=4), dict(seq_len=0),
                dict(workspace=ctypes.c_void_p(12)), dict(grad=q), dict(coef=null), dict(old=null), dict(stats=null)):
        assert pl(**bad) == -1, bad
    lg = lambda **k: lib.slayer_b200_logit_grad(*{**dict(  # noqa: E731
        grad=p, logits=q, dtype=0, action=p, mask=null, stats=p, coef=null, coef_len=1, up=p, up_rows=0, only=0, rows=2, V=5, stride=5, scale=1.0,
        stream=null), **k}.values())
    for bad in (dict(grad=q), dict(stats=null), dict(up=null), dict(coef_len=0)):
        assert lg(**bad) == -1, bad
    pr = lambda **k: lib.slayer_b200_preference_loss(*{**dict(  # noqa: E731
        loss=p, coef=p, workspace=p, logp=p, ref=p, pairs=p, S=2, L=3, P=1, beta=0.1, smoothing=0.0, reduction=0, stream=null), **k}.values())
    for bad in (dict(S=-1), dict(P=-1), dict(L=-1), dict(reduction=2), dict(smoothing=1.1), dict(loss=null), dict(coef=null), dict(pairs=null),
                dict(workspace=ctypes.c_void_p(12))):
        assert pr(**bad) == -1, bad
    assert lib.slayer_b200_policy_loss_workspace(10, 5) >= 88 and lib.slayer_b200_preference_loss_workspace(3) >= 24
