"""CPU: calls of the losses' C entries that would read behind their arrays, or whose numbers the kernels cannot hold."""
import ctypes

from slayerpytorch_b200 import capi

null, p, q = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(32)


def log_prob(**k):
    return capi.load().slayer_b200_log_prob(*{**dict(logp=p, stats=null, logits=q, dtype=0, action=p, mask=null, rows=2, V=5, stride=5, scale=1.0,
                                                     stream=null), **k}.values())


def logit_grad(**k):
    return capi.load().slayer_b200_logit_grad(*{**dict(grad=p, logits=q, dtype=0, action=p, mask=null, stats=p, coef=p, coef_len=1, up=p, up_rows=0,
                                                       only=0, rows=6, V=5, stride=5, scale=1.0, stream=null), **k}.values())


def policy_loss(**k):
    return capi.load().slayer_b200_policy_loss(*{**dict(
        loss=p, grad=null, logp=null, stats=p, coef=p, workspace=p, logits=q, dtype=0, action=p, old=p, adv=p, adv_len=1, ref=null, mask=null,
        rows=6, seq_len=3, V=5, stride=5, scale=1.0, lo=0.2, hi=0.2, kl=0.0, reduction=0, stream=null), **k}.values())


def test_groups_of_rows_are_whole():
    """rows / len values are all there is: a last group that is cut off, or one longer than the rows, has none."""
    for length in (4, 5, 7, 1 << 32, 1 << 40):
        assert logit_grad(coef_len=length) == -1, length
        assert b"whole groups" in capi.load().slayer_b200_last_error()
        assert policy_loss(adv_len=length) == -1, length
        assert b"whole groups" in capi.load().slayer_b200_last_error()


def test_scales_that_no_power_of_two_can_hold():
    """scale * log2(e) is a float32 that is neither infinite nor flushed to zero."""
    for scale in (2.4e38, 3.4e38, 1e-39, 1e-45):
        for call in (log_prob, logit_grad, policy_loss):
            assert call(scale=scale) == -1, scale
            assert b"scale" in capi.load().slayer_b200_last_error()


def test_places_that_the_kernels_cannot_access():
    """Stats are read and written in pairs of floats, logits and gradients by their elements."""
    at = ctypes.c_void_p
    for call in (log_prob, logit_grad, policy_loss):
        for bad in (dict(stats=at(20)), dict(logits=at(34)), dict(logits=at(33), dtype=1), dict(logits=at(33), dtype=2)):
            assert call(**bad) == -1, bad
            assert b"aligned" in capi.load().slayer_b200_last_error()
    for call in (logit_grad, policy_loss):
        for bad in (dict(grad=at(18)), dict(grad=at(17), dtype=1)):
            assert call(**bad) == -1, bad
            assert b"aligned" in capi.load().slayer_b200_last_error()
