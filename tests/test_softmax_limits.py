"""Sizes that the softmax loss refuses before any GPU work (no GPU here)."""
import ctypes as C

from surfface_hip import _lib as E


def test_copies_that_one_launch_does_not_make_are_refused():
    """More than 128 GB to copy (queries; items whose rows start off 16-byte borders): MN_ENOTSUP, not a launch error."""
    need = C.c_size_t()
    w = lambda t, v, d, ty, bwd=1: E.lib().mn_softmax_workspace(t, v, d, ty, bwd, C.byref(need))
    F32, BF16 = E.MN_F32, E.MN_BF16
    assert w(2 ** 24, 1, 1024, BF16) == w(2 ** 24, 1, 2048, F32) == E.MN_OK
    assert w(2 ** 24, 1, 65536, BF16) == w(2 ** 24, 1, 2080, F32) == E.MN_ENOTSUP
    assert w(1, 2 ** 30 - 1, 33, BF16, 0) == w(1, 2 ** 29 - 1, 33, F32, 0) == E.MN_OK
    assert w(1, 2 ** 30, 33, BF16, 0) == w(1, 2 ** 29, 33, F32, 0) == E.MN_ENOTSUP
    assert w(1, 2 ** 31 - 2000, 64, BF16, 0) == E.MN_OK  # rows on borders are not copied
