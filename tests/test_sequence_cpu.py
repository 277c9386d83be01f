"""CPU: what the gated leak and the tensors in 8 bits refuse, and what their C entries do before they touch a GPU."""
import ctypes

import pytest
import torch

from slayerpytorch_b200 import capi, checkpoint, layer
from slayerpytorch_b200.recurrence import gatedLeak, gatedLeakStep

null, p = ctypes.c_void_p(0), ctypes.c_void_p(256)


def test_cpu_tensors_and_options_are_refused():
    x, h = torch.zeros(2, 3, 5), torch.zeros(2, 3)
    for call in (lambda: gatedLeak(x, x), lambda: gatedLeakStep(h, h, h), lambda: checkpoint.compress(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    kept = checkpoint.Checkpoint(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6, 1, dtype=torch.uint8), x.shape, x.dtype)
    for call in (kept.restore, lambda: checkpoint.spikeGrad(x, kept, 1.0, 1.0, 1.0), lambda: checkpoint.weightGrad(x, kept)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for call in (lambda: gatedLeak(x, x, kind="other"), lambda: gatedLeakStep(h, h, h, kind=None)):
        with pytest.raises(ValueError, match="kind"):
            call()
    with pytest.raises(ValueError, match="shape of what was compressed"):
        checkpoint.spikeGrad(x[:1], kept, 1.0, 1.0, 1.0)


def test_layers():
    net = layer.spikeLayer({"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1},
                           {"Ts": 1.0, "tSample": 30})
    assert net.leak(7).gate.shape == (7, 1, 1, 1) and net.leak((4, 5, 3)).gate.shape == (4, 5, 3, 1)
    with pytest.raises(Exception, match="inputSize"):
        net.leak((4, 5))
    assert net.dense(5, 4, checkpoint=True).checkpoint and not net.dense(5, 4).checkpoint
    with pytest.raises(ValueError, match="inputs of its own size"):
        net.dense((4, 4, 2), 3, checkpoint=True)(torch.zeros(1, 2, 5, 4, 6))
    old = net.dense(5, 4)
    del old.__dict__["checkpoint"]      # saved whole before layers had it
    assert old(torch.zeros(1, 5, 1, 1, 6)).shape == (1, 4, 1, 1, 6)


def test_c_entries_of_the_leak():
    lib = capi.load()
    good = dict(y=p, state=null, starts=null, x=p, gate=p, initial=null, dtype=0, flags=0, rows=4, T=10, lengths=null, sample_rows=0, inner=0, period=0,
                workspace=p, stream=null)
    call = lambda **k: lib.slayer_b200_leak_forward(*{**good, **k}.values())  # noqa: E731
    odd = ctypes.c_void_p(257)
    for bad in (dict(dtype=3), dict(flags=4), dict(rows=-1), dict(T=-1), dict(rows=1 << 41), dict(T=1 << 41), dict(rows=1 << 40, T=1 << 40), dict(y=null),
                dict(x=null), dict(gate=null), dict(period=-1), dict(period=2, inner=0), dict(period=3, inner=1), dict(period=8, inner=1),
                dict(period=2, inner=4), dict(lengths=p), dict(x=odd), dict(y=odd), dict(gate=odd), dict(state=odd), dict(starts=odd), dict(initial=odd),
                dict(lengths=ctypes.c_void_p(260), sample_rows=1), dict(T=100000, workspace=null), dict(T=100000, workspace=ctypes.c_void_p(264)),
                dict(rows=1 << 39, T=8)):
        assert call(**bad) == -1, bad
        assert lib.slayer_b200_last_error()
    assert call(rows=0, x=null, y=null, gate=null) == 0
    good = dict(dx=p, dgate=p, dinitial=null, g=p, gstate=null, starts=p, x=p, gate=p, dtype=0, flags=0, rows=4, T=10, lengths=null, sample_rows=0, inner=0,
                period=0, workspace=p, stream=null)
    call = lambda **k: lib.slayer_b200_leak_backward(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=-1), dict(g=null), dict(starts=null), dict(dx=odd), dict(dgate=odd), dict(g=odd), dict(gstate=odd), dict(dinitial=odd),
                dict(period=2, inner=2, workspace=null), dict(T=100000, workspace=null)):
        assert call(**bad) == -1, bad
    assert call(rows=0, x=null, g=null, gate=null, starts=null) == 0
    good = dict(y=p, state=p, x=p, gate=p, dtype=1, gate_dtype=1, flags=0, rows=4, inner=0, period=0, stream=null)
    call = lambda **k: lib.slayer_b200_leak_step(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=3), dict(gate_dtype=2), dict(state=null), dict(y=null), dict(x=odd), dict(state=ctypes.c_void_p(258)), dict(rows=-1),
                dict(period=3, inner=1)):
        assert call(**bad) == -1, bad
    assert call(rows=0, y=null) == 0
    # a state for each lane: of 4, 8 or 16 steps (up to 16 of them), else of 12 or 16, with up to three before the first one
    for T, n in ((0, 0), (1, 1), (4, 1), (5, 1), (16, 1), (17, 2), (128, 8), (129, 16), (300, 32), (509, 32), (511, 64), (512, 32), (513, 64), (1450, 96),
                 (2000, 128), (100000, 196 * 32)):
        assert lib.slayer_b200_leak_states(T) == n, T
    assert lib.slayer_b200_leak_states(-1) == -1 and lib.slayer_b200_leak_states(1 << 31) == -1
    assert lib.slayer_b200_leak_workspace(-1, 5, 0, 0, 0) == -1
    assert lib.slayer_b200_leak_workspace(1 << 20, 300, 0, 0, 0) == 0


def test_c_entries_of_tensors_in_8_bits():
    lib = capi.load()
    odd = ctypes.c_void_p(257)
    good = dict(q=p, scale=p, x=p, dtype=0, rows=4, T=10, stream=null)
    call = lambda **k: lib.slayer_b200_compress8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=3), dict(rows=-1), dict(T=-1), dict(rows=1 << 41), dict(rows=1 << 39, T=64), dict(q=null), dict(scale=null), dict(x=null),
                dict(q=odd), dict(x=odd)):
        assert call(**bad) == -1, bad
        assert lib.slayer_b200_last_error()
    assert call(rows=0, q=null) == 0 and call(T=0, x=null) == 0
    good = dict(out=p, q=p, scale=p, dtype=0, rows=4, T=10, stream=null)
    call = lambda **k: lib.slayer_b200_restore8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=3), dict(rows=-1), dict(q=null), dict(scale=null), dict(out=null), dict(q=odd), dict(out=odd)):
        assert call(**bad) == -1, bad
    good = dict(out=p, g=p, q=p, scale_bytes=p, rows=4, T=10, theta=1.0, tau=1.0, scale=1.0, stream=null)
    call = lambda **k: lib.slayer_b200_spike_grad8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(rows=-1), dict(q=null), dict(scale_bytes=null), dict(out=null), dict(g=null), dict(q=odd), dict(g=odd)):
        assert call(**bad) == -1, bad
    good = dict(out=p, g=p, q=p, scale=p, N=2, O=3, I=4, T=5, workspace=p, stream=null)
    call = lambda **k: lib.slayer_b200_weight_grad8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(N=-1), dict(O=-1), dict(I=-1), dict(T=-1), dict(N=1 << 32), dict(O=1 << 30), dict(I=1 << 32), dict(T=1 << 32), dict(out=null), dict(g=null),
                dict(q=null), dict(scale=null), dict(q=odd), dict(g=odd), dict(out=odd), dict(N=900, T=300, workspace=null)):
        assert call(**bad) == -1, bad
    assert call(O=0, out=null) == 0 and call(I=0, out=null) == 0
    assert lib.slayer_b200_weight_grad8_workspace(-1, 2, 3, 4) == -1 and lib.slayer_b200_weight_grad8_workspace(0, 2, 3, 4) == 0
