"""CPU: what the orthogonalised updates refuse, and what their C entries do before they touch a GPU."""
import ctypes

import pytest
import torch

from slayerpytorch_b200 import capi, optim


def test_lists_shapes_and_options_are_checked():
    w, g, m = torch.zeros(4, 5), torch.zeros(4, 5), torch.zeros(4, 5)
    for bad in (dict(grads=[]), dict(momenta=[m, m]), dict(weights=[w[0]]), dict(adjust="other"), dict(momenta=[torch.zeros(5, 4).t()]),
                dict(weights=[w, w], grads=[g, g], momenta=[m, m.clone()]), dict(weights=[w, w + 1], grads=[g, g], momenta=[m, m])):
        with pytest.raises(ValueError):
            optim.muonStep(**{**dict(weights=[w], grads=[g], momenta=[m], lr=0.1), **bad})
    with pytest.raises(ValueError, match="in the memory of"):
        optim.muonStep([w], [m], [m], lr=0.1)
    with pytest.raises(ValueError, match="sparse"):
        optim.muonStep([w], [g.to_sparse()], [m], lr=0.1)
    with pytest.raises(ValueError, match="two dimensions"):
        optim.orthogonalize(w[0])
    with pytest.raises(ValueError, match="no gradient"):
        optim.orthogonalize(w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.orthogonalize(w)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.muonStep([w], [g], [m], lr=0.1)
    optim.muonStep([], [], [], lr=0.1)
    p = torch.nn.Parameter(w.clone())
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weightDecay=-0.1), dict(adjust="other")):
        with pytest.raises(ValueError):
            optim.Muon([p], **bad)
    with pytest.raises(ValueError, match="two dimensions"):
        optim.Muon([p, torch.nn.Parameter(torch.zeros(3))])


def test_c_entries_check_their_arguments():
    lib = capi.load()
    null, p = ctypes.c_void_p(0), ctypes.c_void_p(256)
    good = dict(out=p, inp=p, dtype=0, batch=1, rows=4, cols=5, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, workspace=p, stream=null)
    call = lambda **k: lib.slayer_b200_orthogonalize(*{**good, **k}.values())  # noqa: E731
    nan, inf = float("nan"), float("inf")
    for bad in (dict(dtype=5), dict(batch=-1), dict(rows=-1), dict(steps=0), dict(steps=101), dict(a=nan), dict(b=inf), dict(c=5.0), dict(a=9.0),
                dict(eps=-1.0), dict(eps=nan), dict(out=null), dict(workspace=null), dict(workspace=ctypes.c_void_p(128))):
        assert call(**bad) == -1, bad
        assert lib.slayer_b200_last_error()
    for far in (dict(rows=33000, cols=33000), dict(rows=1, cols=1 << 23), dict(rows=1 << 40, cols=1 << 40)):
        assert call(**far) == -3, far
    assert call(batch=0, inp=null, out=null, workspace=null) == 0
    lst = (capi.MuonMatrix * 2)()
    for i in range(2):
        lst[i].weight = lst[i].grad = lst[i].momentum = 256
        lst[i].rows, lst[i].cols = 4, 5
    step = dict(lst=ctypes.cast(lst, ctypes.c_void_p), count=2, dtype=0, lr=0.1, mu=0.9, nesterov=1, decay=0.0, adjust=1, steps=5, a=3.4445, b=-4.775,
                c=2.0315, eps=1e-7, workspace=p, stream=null)
    call = lambda **k: lib.slayer_b200_muon_step(*{**step, **k}.values())  # noqa: E731
    for bad in (dict(dtype=3), dict(count=-1), dict(lst=null), dict(adjust=3), dict(steps=0), dict(workspace=null), dict(workspace=ctypes.c_void_p(8))):
        assert call(**bad) == -1, bad
    lst[1].momentum = None
    assert call() == -1
    lst[1].momentum, lst[1].rows = 256, -1
    assert call() == -1
    lst[0].rows = lst[1].rows = 0
    assert call(workspace=null) == 0
    assert call(count=0, lst=null, workspace=null) == 0
    lst[0].rows, lst[0].cols = 30, 20
    assert lib.slayer_b200_muon_step_workspace(step["lst"], 2, 0) >= lib.slayer_b200_orthogonalize_workspace(1, 30, 20, 0) > 0
    assert lib.slayer_b200_orthogonalize_workspace(0, 30, 20, 0) == 0
