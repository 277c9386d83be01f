"""CPU: sizes that the orthogonalised updates refuse have no workspace."""
import ctypes

from slayerpytorch_b200 import capi


def test_matrices_that_are_too_large_have_no_workspace():
    lib = capi.load()
    lst = (capi.MuonMatrix * 2)()
    for m in lst:
        m.weight = m.grad = m.momentum = 256
        m.rows, m.cols = 4, 5
    for rows, cols in ((33000, 33000), (1, (1 << 22) + 1), ((1 << 22) + 1, 1), (1 << 40, 1 << 40), (32768, 65537)):
        assert lib.slayer_b200_orthogonalize_workspace(1, rows, cols, 0) == -3
        assert b"a matrix of" in lib.slayer_b200_last_error()
        lst[1].rows, lst[1].cols = rows, cols
        assert lib.slayer_b200_muon_step_workspace(ctypes.cast(lst, ctypes.c_void_p), 2, 0) == -3
    lst[1].rows, lst[1].cols = 1, 1 << 22
    assert lib.slayer_b200_orthogonalize_workspace(1, 1, 1 << 22, 0) > 0
    assert lib.slayer_b200_muon_step_workspace(ctypes.cast(lst, ctypes.c_void_p), 2, 0) > 0
