"""Argument checks of the item scores and the softmax loss at the C entries:
every bad call is refused before any GPU work (no GPU here)."""
import ctypes as C

import pytest
import torch

import surfface_hip as S
from surfface_hip import _lib

A = C.c_void_p(4096)      # never read: every call below is refused first
ODD = C.c_void_p(4100)
E = _lib


def test_quantize_and_dequantize_refusals():
    L = E.lib()
    q = lambda X=A, ty=0, n=4, d=20, codes=A, ld=32, s=A: L.mn_quantize_rows_i8(X, ty, n, d, codes, ld, s, None)
    dq = lambda codes=A, ld=32, s=A, n=4, d=20, X=A, ty=0: L.mn_dequantize_rows_i8(codes, ld, s, n, d, X, ty, None)
    for f in (q, dq):
        assert f(n=-1) == E.MN_EINVAL and f(d=0) == E.MN_EINVAL and f(ld=16) == E.MN_EINVAL
        assert f(ld=40) == E.MN_EINVAL and f(ld=1 << 32) == E.MN_EINVAL and f(ld=2 ** 31 - 16) == E.MN_EINVAL
        assert f(ty=1) == E.MN_ENOTSUP and f(ty=7) == E.MN_ENOTSUP
        assert f(X=None) == E.MN_EINVAL and f(codes=None) == E.MN_EINVAL and f(s=None) == E.MN_EINVAL
        assert f(codes=ODD) == E.MN_EINVAL
        assert f(n=0) == E.MN_OK
    assert b"" == L.mn_last_error()


def test_scores_refusals():
    L = E.lib()

    def f(Q=A, ldq=32, qs=A, m=4, c=A, ldc=32, cs=A, n=9, d=20, Y=A, ty=0, ws=A, wb=1 << 20):
        return L.mn_scores_i8(Q, ldq, qs, m, c, ldc, cs, n, d, Y, ty, ws, wb, None)

    assert f(m=-1) == f(n=-1) == f(d=0) == E.MN_EINVAL
    assert f(d=131072, ldq=131072, ldc=131072) == E.MN_ENOTSUP
    assert f(ldq=16) == f(ldc=16) == f(ldq=24) == f(ldc=40) == E.MN_EINVAL
    assert f(ty=1) == f(ldq=(1 << 23) + 16) == f(ldc=1 << 40) == E.MN_ENOTSUP
    assert f(Q=None) == f(c=None) == f(qs=None) == f(cs=None) == f(Y=None) == E.MN_EINVAL
    assert f(Q=ODD) == f(c=ODD) == E.MN_EINVAL
    assert f(m=65, ws=None) == f(m=65, wb=65 * 64 - 1) == f(m=65, ws=ODD) == E.MN_ECAP
    assert f(m=0) == f(n=0) == E.MN_OK
    b = C.c_size_t()
    assert L.mn_scores_i8_workspace(65, 20, C.byref(b)) == 0 and b.value == 65 * 64
    assert L.mn_scores_i8_workspace(64, 20, C.byref(b)) == 0 and b.value == 0
    assert L.mn_scores_i8_workspace(64, 131071, C.byref(b)) == 0 and b.value == 64 * 131072
    assert L.mn_scores_i8_workspace(65, 128, C.byref(b)) == 0 and b.value == 0
    assert L.mn_scores_i8_workspace(4, 131072, C.byref(b)) == E.MN_EINVAL
    assert L.mn_scores_i8_workspace(4, 20, None) == E.MN_EINVAL


def test_softmax_refusals():
    L = E.lib()
    need = C.c_size_t()
    for bwd in (0, 1):
        assert L.mn_softmax_workspace(4, 9, 20, 0, bwd, C.byref(need)) == 0 and need.value > 0
        assert L.mn_softmax_workspace(0, 9, 20, 0, bwd, C.byref(need)) == 0 and need.value == 0
    assert L.mn_softmax_workspace(4, 9, 20, 0, 0, None) == E.MN_EINVAL

    def st(Q=A, c=A, ty=0, t=4, v=9, d=20, at=A, off=0, s=1.0, rest=A, zt=A, loss=A, mean=A, share=A, ws=A,
           wb=1 << 30):
        return L.mn_softmax_stats(Q, c, ty, t, v, d, at, off, s, rest, zt, loss, mean, share, ws, wb, None)

    def bw(Q=A, c=A, ty=0, t=4, v=9, d=20, at=A, off=0, s=1.0, rest=A, zt=A, g=A, gn=1, gs=A, dq=A, dc=A, ws=A,
           wb=1 << 40):
        return L.mn_softmax_backward(Q, c, ty, t, v, d, at, off, s, rest, zt, g, gn, gs, dq, dc, ws, wb, None)

    for f in (st, bw):
        assert f(t=-1) == f(v=0) == f(d=0) == f(off=-1) == E.MN_EINVAL
        assert f(s=0.0) == f(s=-2.0) == f(s=float("nan")) == f(s=float("inf")) == E.MN_EINVAL
        assert f(ty=1) == f(ty=5) == E.MN_ENOTSUP
        assert f(v=2 ** 31 - 1) == f(t=2 ** 24 + 1) == f(d=65537) == f(t=2 ** 24, v=2 ** 31 - 2000) == E.MN_ENOTSUP
        assert f(Q=None) == f(c=None) == f(at=None) == f(rest=None) == f(zt=None) == E.MN_EINVAL
        assert f(Q=ODD) == f(c=ODD) == E.MN_EINVAL
        assert f(ws=None) == f(wb=100) == f(ws=ODD) == E.MN_ECAP
    assert st(loss=None) == st(share=None) == E.MN_EINVAL
    assert bw(gn=3) == bw(g=None) == bw(dq=None, dc=None) == bw(t=0) == E.MN_EINVAL

    def mg(r=A, z=A, p=2, t=4, at=A, rest=A, zt=A, loss=A, mean=A, share=A):
        return L.mn_softmax_merge(r, z, p, t, at, rest, zt, loss, mean, share, None)

    assert mg(p=0) == mg(t=-1) == mg(r=None) == mg(z=None) == mg(at=None) == mg(rest=None) == E.MN_EINVAL
    assert mg(loss=None) == mg(share=None) == mg(zt=None) == mg(t=2 ** 24 + 1) == E.MN_EINVAL


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 16)
    for f in (lambda: S.quantize_rows(x), lambda: S.softmax_loss(x, x, torch.zeros(4).long()),
              lambda: S.softmax_stats(x, x, torch.zeros(4).long()),
              lambda: S.scores_i8(S.Int8Rows(x.char(), x[:, 0], 16), S.Int8Rows(x.char(), x[:, 0], 16)),
              lambda: S.dequantize_rows(S.Int8Rows(x.char(), x[:, 0], 16))):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(ValueError):
        S.softmax_loss(x, x, torch.zeros(4).long(), reduction="max")
