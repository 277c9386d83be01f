"""CPU: what the C entries of the gated leak may write over.  (Nothing here is launched: all calls are refused.)"""
import ctypes

import pytest

from slayerpytorch_b200 import capi

R, T, E = 6, 40, 4
ALL, ROWS = R * T * E, R * 4
AT = {name: (i + 1) << 20 for i, name in enumerate(("y", "state", "starts", "workspace", "x", "gate", "initial", "lengths", "dx", "dgate", "dinitial", "g", "gstate"))}


def refused(entry, args, **moved):
    args = {**args, **moved}
    rc = getattr(capi.load(), "slayer_b200_leak_" + entry)(*(v if k in ("dtype", "gate_dtype", "flags", "rows", "T", "sample_rows", "inner", "period")
                                                             else ctypes.c_void_p(v) for k, v in args.items()))
    assert rc == -1
    return b"share" in capi.load().slayer_b200_last_error()


FORWARD = dict(y=AT["y"], state=AT["state"], starts=AT["starts"], x=AT["x"], gate=AT["gate"], initial=AT["initial"], dtype=0, flags=0, rows=R, T=T,
               lengths=AT["lengths"], sample_rows=2, inner=0, period=0, workspace=AT["workspace"], stream=0)
BACKWARD = dict(dx=AT["dx"], dgate=AT["dgate"], dinitial=AT["dinitial"], g=AT["g"], gstate=AT["gstate"], starts=AT["starts"], x=AT["x"], gate=AT["gate"], dtype=0,
                flags=0, rows=R, T=T, lengths=AT["lengths"], sample_rows=2, inner=0, period=0, workspace=AT["workspace"], stream=0)


@pytest.mark.parametrize("name,other,by", [("y", "x", 0), ("y", "x", ALL - 16), ("x", "y", 16), ("y", "gate", 0), ("y", "initial", 0), ("y", "starts", 0),
                                           ("y", "state", 0), ("state", "initial", 4), ("initial", "state", ROWS - 4), ("state", "x", 8), ("state", "lengths", 20),
                                           ("starts", "state", 0), ("starts", "gate", ALL - 4), ("lengths", "y", ALL - 8)])
def test_forward(name, other, by):
    assert refused("forward", FORWARD, **{name: AT[other] + by})


@pytest.mark.parametrize("name,other,by", [("dx", "g", 0), ("dx", "x", 0), ("dgate", "gate", 0), ("dgate", "dx", ALL - 16), ("dx", "dgate", ALL - 16), ("dgate", "g", 16),
                                           ("dinitial", "gstate", 4), ("gstate", "dinitial", ROWS - 4), ("dinitial", "dx", 0), ("dinitial", "starts", 0),
                                           ("dx", "starts", 0), ("dinitial", "lengths", 20)])
def test_backward(name, other, by):
    assert refused("backward", BACKWARD, **{name: AT[other] + by})


def test_workspaces():
    """Of rows that are split (1000000 steps), and of a gate per row."""
    size = capi.load().slayer_b200_leak_workspace(R, 1000000, 0, 0, 0)
    assert size > 16
    far = {name: (i + 1) << 30 for i, name in enumerate(AT)}
    for entry, args in (("forward", FORWARD), ("backward", BACKWARD)):
        args = {k: far.get(k, v) for k, v in args.items()}
        for other in ("x", "gate", "starts", "state" if entry == "forward" else "dinitial"):
            assert refused(entry, args, T=1000000, workspace=far[other])
    assert refused("backward", BACKWARD, inner=1, period=R, workspace=AT["g"])
    assert refused("backward", BACKWARD, inner=1, period=R, workspace=AT["dgate"])


def test_step():
    good = dict(y=AT["y"], state=AT["state"], x=AT["x"], gate=AT["gate"], dtype=0, gate_dtype=0, flags=0, rows=R, inner=0, period=0, stream=0)
    for moved in (dict(state=AT["x"]), dict(state=AT["gate"] + 20), dict(state=AT["y"] - 20), dict(y=AT["x"] + 4), dict(y=AT["x"] - 4), dict(y=AT["gate"] + 4),
                  dict(y=AT["gate"], inner=1, period=3), dict(y=AT["gate"], dtype=1)):
        assert refused("step", good, **moved)
