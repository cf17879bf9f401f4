"""Refusals, workspaces and shape propagation of the dense layer and the distillation loss: host
logic that runs before any launch (no GPU, no pointer is followed)."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(17)


@pytest.fixture(scope="module")
def L():
    from objectdetection_amd import _lib
    return _lib


def fwd(L, x=ONE, ldx=64, w=ONE, ldw=32, layout=0, bias=None, res=None, ldr=0, M=4, K=64, N=32, dt=2, act=0,
        out=ONE, ldo=32, odt=2, pre=None, ldp=0, ws=None, wsb=0):
    return L.lib.frcnn_dense_fwd(x, ldx, w, ldw, layout, bias, res, ldr, M, K, N, dt, act, out, ldo, odt, pre, ldp,
                                 ws, wsb, None)


def bwd(L, d=ONE, ldd=32, ddt=2, x=ONE, ldx=64, w=ONE, ldw=32, layout=0, pre=None, ldp=0, M=4, K=64, N=32, dt=2,
        act=0, dx=ONE, lddx=64, dw=ONE, lddw=32, db=ONE, ws=ONE, wsb=1 << 40):
    return L.lib.frcnn_dense_bwd(d, ldd, ddt, x, ldx, w, ldw, layout, pre, ldp, M, K, N, dt, act, dx, lddx, dw, lddw,
                                 db, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(out=None), dict(ldx=63), dict(ldw=31), dict(layout=1, ldw=63), dict(layout=2),
    dict(ldo=31), dict(M=-1), dict(K=0), dict(N=0), dict(dt=0), dict(dt=3), dict(act=-1), dict(act=4), dict(odt=1),
    dict(res=ONE, ldr=31), dict(pre=ONE, ldp=31), dict(x=ODD), dict(out=ctypes.c_void_p(18), odt=0), dict(bias=ODD)])
def test_dense_forward_refuses(L, bad):
    assert fwd(L, **bad) == L.E_BADARG


@pytest.mark.parametrize("bad", [
    dict(d=None), dict(ldd=31), dict(ddt=1), dict(dx=None, dw=None, db=None), dict(w=None), dict(x=None),
    dict(lddx=63), dict(lddw=31), dict(layout=1, lddw=63), dict(act=1), dict(act=2, pre=ONE, ldp=31), dict(dt=0),
    dict(M=-1), dict(K=0), dict(N=0), dict(d=ctypes.c_void_p(18), ddt=0), dict(db=ODD)])
def test_dense_backward_refuses(L, bad):
    assert bwd(L, **bad) == L.E_BADARG


def test_dense_workspaces(L):
    f, b = L.lib.frcnn_dense_fwd_workspace_bytes, L.lib.frcnn_dense_bwd_workspace_bytes
    assert f(0, 8, 8, 0, 0) == 0 and b(0, 8, 8, 0, 0) == 0 and f(4, 0, 8, 0, 0) == 0 and f(-1, 8, 8, 0, 0) == 0
    assert f(16000, 4096, 4096, 0, 3) == 0                 # enough tiles: no split; aligned: no copy
    copy = lambda rows, cols: (rows * ((cols + 7) // 8) * 16 + 255) // 256 * 256
    assert f(16000, 4096, 4096, 0, 2) == copy(16000, 4096) and f(16000, 4096, 4096, 1, 1) == copy(4096, 4096)
    assert f(16000, 4095, 4096, 0, 3) == copy(16000, 4095)
    assert f(16000, 4095, 4095, 0, 0) == copy(16000, 4095) + copy(4095, 4095)
    for layout, ldw in ((0, 64), (1, 25088)):
        need = f(2, 25088, 64, layout, 0)
        assert need > 0 and need == f(2, 25088, 64, layout, 3)     # few rows: partial sums, no copy
        small = dict(M=2, K=25088, ldx=25088, N=64, layout=layout, ldw=ldw, ldo=64)
        assert fwd(L, **small) == L.E_WORKSPACE and fwd(L, ws=ONE, wsb=need - 1, **small) == L.E_WORKSPACE
    odd = dict(M=100, ldx=65)                              # a stride that is no multiple of 8: x is copied
    assert fwd(L, ws=ONE, wsb=f(100, 64, 32, 0, 2) - 1, **odd) == L.E_WORKSPACE
    assert b(100, 64, 32, 0, 0) >= 100 * 32 * 2 + copy(100, 64)
    assert b(100, 64, 33, 0, 3) - b(100, 64, 33, 0, 1) == copy(64, 33) * 0      # 33: W is copied either way
    assert b(100, 64, 32, 0, 7) < b(100, 64, 32, 0, 3) <= b(100, 64, 32, 0, 0)
    relu = dict(act=1, pre=ONE, ldp=32)                    # dz is kept in the workspace
    assert bwd(L, ws=None, **relu) == L.E_WORKSPACE
    assert bwd(L, wsb=b(4, 64, 32, 0, 3) - 1, **relu) == L.E_WORKSPACE
    assert bwd(L, ws=ctypes.c_void_p(24), **relu) == L.E_WORKSPACE
    wide = (1 << 21) + 8                                    # rows that a tile cannot reach over
    assert fwd(L, M=40, K=wide, ldx=wide, ws=ONE, wsb=1 << 50) == L.E_UNSUPPORTED
    assert bwd(L, M=40, N=wide, ldd=wide, ldw=wide, lddw=wide, ws=ONE, wsb=1 << 50) == L.E_UNSUPPORTED
    assert fwd(L, M=1 << 31) == L.E_UNSUPPORTED and bwd(L, M=1 << 31) == L.E_UNSUPPORTED
    assert fwd(L, M=0, x=None, out=None) == L.OK           # no rows: nothing to do, nothing launched


def loss(L, z=ONE, ldz=50, dt=0, t=ONE, tdt=0, idx=ONE, w=None, rows=3, V=50, k=4, T=1.0, g=1.0, l=ONE, lse=ONE,
         d=None, ldg=50, ws=None, wsb=0):
    return L.lib.frcnn_distill_loss(z, ldz, dt, t, tdt, idx, w, rows, V, k, T, g, l, lse, d, ldg, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(z=None), dict(t=None), dict(idx=None), dict(l=None), dict(lse=None), dict(ldz=49), dict(d=ONE, ldg=49),
    dict(dt=3), dict(tdt=1), dict(rows=-1), dict(V=0), dict(k=0), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")),
    dict(T=float("inf")), dict(T=1e-19), dict(T=1e19), dict(z=ctypes.c_void_p(18)), dict(idx=ctypes.c_void_p(20))])
def test_distillation_refuses(L, bad):
    assert loss(L, **bad) == L.E_BADARG
    b = dict(z=ONE, ldz=50, dt=0, t=ONE, tdt=0, idx=ONE, lse=ONE, w=None, rows=3, V=50, k=4, T=1.0, d=ONE, ldg=50)
    bad = {k: v for k, v in bad.items() if k in b}
    if not bad:
        bad = dict(lse=None)
    b.update(bad)
    assert L.lib.frcnn_distill_bwd(ONE, b["z"], b["ldz"], b["dt"], b["t"], b["tdt"], b["idx"], b["lse"], b["w"],
                                   b["rows"], b["V"], b["k"], b["T"], b["d"], b["ldg"], None) == L.E_BADARG


def test_distillation_limits(L):
    assert loss(L, k=L.DISTILL_MAX_K + 1) == L.E_UNSUPPORTED
    need = L.lib.frcnn_distill_workspace_bytes
    assert need(128000, 21, 8, 0) == 0 and need(4096, 65536, 64, 2) == 0 and need(0, 1 << 20, 8, 0) == 0
    big = need(1, 131072, 64, 0)
    assert big > 0
    wide = dict(rows=1, V=131072, k=64, ldz=131072)
    assert loss(L, **wide) == L.E_WORKSPACE and loss(L, ws=ONE, wsb=big - 1, **wide) == L.E_WORKSPACE
    assert loss(L, ws=ctypes.c_void_p(20), wsb=big, **wide) == L.E_WORKSPACE
    assert loss(L, rows=0, z=None, t=None, idx=None) == L.OK


def test_cpu_tensors_are_refused():
    from objectdetection_amd import ops
    x = torch.zeros((2, 8), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.dense_fwd(x, torch.zeros((8, 4), dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        ops.distill_loss(torch.zeros((2, 8)), torch.zeros((2, 3)), torch.zeros((2, 3), dtype=torch.int64))


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from objectdetection_amd import torch_ops  # noqa: F401
    F = torch.ops.frcnn
    with FakeTensorMode():
        e = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="cuda")
        w = e(96, 392).t().requires_grad_(True)
        out, pre = F.dense(e(2, 5, 7, 7, 8), w, e(96), e(2, 5, 96), "relu", True)
        assert out.shape == (2, 5, 96) and pre.shape == out.shape and out.requires_grad and not pre.requires_grad
        assert F.dense(e(4, 392), w, None, None, "none", False)[1].shape == (0,)
        dx, dw, db = F.dense_backward(out, e(2, 5, 7, 7, 8), w, pre, "relu")
        assert dx.shape == (2, 5, 7, 7, 8) and dw.shape == (392, 96) and dw.stride() == (1, 392) and db.shape == (96,)
        z = e(2, 5, 21, dt=torch.float32).requires_grad_(True)
        t, i = e(2, 5, 8, dt=torch.float32), e(2, 5, 8, dt=torch.int64)
        loss, lse = F.distill_loss(z, t, i, None, 2.0)
        assert loss.shape == (2, 5) and loss.requires_grad and lse.shape == (2, 5) and not lse.requires_grad
        assert F.distill_loss_backward(loss, z, t, i, lse, None, 2.0).shape == z.shape


def test_head_dtype_is_checked():
    from objectdetection_amd.train import FRCNModel
    with pytest.raises(ValueError):
        FRCNModel(8, 7, 16, 21, dtype=torch.float64)
    m, n = FRCNModel(8, 7, 16, 21), FRCNModel(8, 7, 16, 21, dtype=torch.bfloat16)
    assert {k: v.shape for k, v in m.state_dict().items()} == {k: v.shape for k, v in n.state_dict().items()}
    assert all(v.dtype == torch.float32 for v in n.state_dict().values())


def test_a_launch_has_fewer_than_2_32_threads(L):
    assert fwd(L, M=(1 << 30) - 63) == L.E_UNSUPPORTED
    far = dict(M=1 << 29, K=67, ldx=67, ws=ONE, wsb=1 << 62)   # 2^32 pieces would be copied
    assert fwd(L, ldw=67, layout=1, **far) == L.E_UNSUPPORTED
    assert bwd(L, ldw=67, layout=1, lddw=67, lddx=67, **far) == L.E_UNSUPPORTED
    assert bwd(L, M=0, K=2097152, N=4096, ldd=4096, ldw=4096, lddx=2097152, lddw=4096) == L.E_UNSUPPORTED


def test_kernels_keep_everything_in_registers():
    """Nothing of the dense and distillation kernels waits in scratch memory, and eight waves of the
    large tile fit on a compute unit (256 registers per lane)."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools"))
    from kernel_budgets import kernel_budgets
    own = {n: k for n, k in kernel_budgets().items() if "dense_" in n or "distill_" in n}
    assert len(own) > 60
    for name, k in own.items():
        assert k["scratch"] == 0 and k["vgpr"] <= (256 if k["wg_max"] <= 512 else 128), (name, k)
