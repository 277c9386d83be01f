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


def test_places_that_the_kernels_cannot_access():
    lib, at = capi.load(), ctypes.c_void_p
    for dtype, off in ((0, 2), (0, 1), (1, 1), (2, 1)):
        for out, src in ((256 + off, 256), (256, 256 + off)):
            assert lib.slayer_b200_orthogonalize(at(out), at(src), dtype, 1, 4, 5, 5, 3.4445, -4.775, 2.0315, 1e-7, at(256), at(0)) == -1
            assert b"aligned" in lib.slayer_b200_last_error()
    for dtype, bad in ((0, dict(weight=258)), (0, dict(grad=258)), (1, dict(weight=257)), (2, dict(grad=257)), (1, dict(momentum=258))):
        m = capi.MuonMatrix(**{**dict(weight=256, grad=256, momentum=256, rows=4, cols=5), **bad})
        assert lib.slayer_b200_muon_step(ctypes.cast(ctypes.pointer(m), at), 1, dtype, 0.1, 0.9, 1, 0.0, 1, 5, 3.4445, -4.775, 2.0315, 1e-7, at(256),
                                         at(0)) == -1
        assert b"aligned" in lib.slayer_b200_last_error()


def test_workspaces_of_many_large_matrices_are_bounded():
    """A stack or a list of large matrices is worked on a few at a time: 4 GB, or what one of them needs."""
    lib = capi.load()
    for side, count in ((4096, 48), (8192, 100), (16384, 25)):
        for dtype in (0, 1, 2):
            one = lib.slayer_b200_orthogonalize_workspace(1, side, side, dtype)
            assert 0 < lib.slayer_b200_orthogonalize_workspace(count, side, side, dtype) <= max(one, 4 << 30)
            lst = (capi.MuonMatrix * (2 * count))()
            for i, m in enumerate(lst):
                m.rows, m.cols = (side, side) if i % 2 else (300, 500)
            assert one <= lib.slayer_b200_muon_step_workspace(ctypes.cast(lst, ctypes.c_void_p), 2 * count, dtype) <= max(one, 4 << 30)
