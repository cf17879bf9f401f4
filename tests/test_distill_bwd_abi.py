"""What the distillation's backward refuses before any launch (no GPU, no pointer is followed)."""
import ctypes

import pytest

ONE = ctypes.c_void_p(16)


@pytest.fixture(scope="module")
def L():
    from objectdetection_amd import _lib
    return _lib


def bwd(L, g=ONE, z=ONE, ldz=131072, dt=0, t=ONE, tdt=0, idx=ONE, lse=ONE, w=None, rows=1, V=131072, k=4, T=1.0, d=ONE, ldg=131072,
        ws=None, wsb=0):
    return L.lib.frcnn_distill_bwd_ws(g, z, ldz, dt, t, tdt, idx, lse, w, rows, V, k, T, d, ldg, ws, wsb, None)


@pytest.mark.parametrize("bad", [dict(g=None), dict(z=None), dict(t=None), dict(idx=None), dict(lse=None), dict(d=None),
                                 dict(ldz=131071), dict(ldg=131071), dict(dt=3), dict(tdt=1), dict(rows=-1), dict(V=0), dict(k=0),
                                 dict(T=0.0), dict(T=float("nan")), dict(z=ctypes.c_void_p(18))])
def test_refuses(L, bad):
    assert bwd(L, **bad) == L.E_BADARG


def test_a_workspace_that_is_given_is_large_enough(L):
    need = L.lib.frcnn_distill_workspace_bytes(1, 131072, 4, 0)
    assert need > 0
    assert bwd(L, ws=ONE, wsb=need - 1) == L.E_WORKSPACE and bwd(L, ws=ctypes.c_void_p(20), wsb=need) == L.E_WORKSPACE
    assert bwd(L, k=L.DISTILL_MAX_K + 1) == L.E_UNSUPPORTED
    assert bwd(L, rows=0, z=None, t=None, idx=None) == L.OK
