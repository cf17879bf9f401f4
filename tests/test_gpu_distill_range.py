"""Distillation of logits whose values over T are large while their differences are not: what a common
offset, a small temperature or masks of the lowest value must not change.

Derived before any run: relative to the row's maximum a difference d of logits is one float32 subtraction and two
roundings of d / T, so a logarithm of a probability is off by at most 2^-21 (|log p| + 8) whatever the logits' own
size (+ the sums of V and k terms, (V / 256 + k + 32) 2^-23 as lanes share them); p and q by as much relative.  Below float32's smallest normal number
an exponential may be 0 (e^(d / T) comes before its factor c = T): with the sum of all of them at least 1, q and each p
of a label are then off by 2^-126, and c q and c p by 2^-126 T, which a large T lifts into sight."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
# a lane per class, several rows a wave, one workgroup a row (with and without the table), two launches, longer than registers
SHAPES = [(40, 8, 5), (300, 21, 8), (60, 1203, 40), (30, 4000, 100), (220, 20003, 12), (3, 40000, 64), (2, 70001, 300), (300, 70001, 6)]


def reference(z, t, idx, T):
    """loss and gradient of loss.sum() with their tolerances, float64."""
    z, t, idx = z.double().cpu(), t.double().cpu(), idx.cpu()
    V, k = z.shape[1], t.shape[1]
    there = (idx >= 0) & (t > -math.inf)
    t = torch.where(there, t, torch.full_like(t, -math.inf))
    log_p = torch.log_softmax((t - t.amax(1, keepdim=True)) / T, 1)
    log_q = torch.log_softmax((z - z.amax(1, keepdim=True)) / T, 1)
    p, q, at = log_p.exp(), log_q.exp(), idx.clamp(min=0)
    lq = log_q.gather(1, at)
    zero = torch.zeros_like(p)
    sums = (V / 256 + k + 32) * 2.0 ** -23
    rp, rq = 2.0 ** -21 * (log_p.abs() + 8) + sums, 2.0 ** -21 * (log_q.abs() + 8) + sums
    rlq = rq.gather(1, at)
    part = p > 0
    loss = T * T * torch.where(part, p * (log_p - lq), zero).sum(1)
    tol_l = T * T * torch.where(part, p * (rp * (1 + (log_p - lq).abs()) + rlq), zero).sum(1)
    full = torch.zeros_like(z).scatter_add_(1, at, torch.where(part, p, zero))
    tol_f = torch.zeros_like(z).scatter_add_(1, at, torch.where(part, p * rp, zero))
    return loss, T * (q - full), 1.01 * tol_l, 1.01 * T * (torch.where(q > 0, q * rq, torch.zeros_like(q)) + tol_f + 2 * 2.0 ** -126)


def make(seed, dev, rows, V, k, spread):
    g = torch.Generator().manual_seed(seed)
    z = spread * torch.randn((rows, V), generator=g)
    t = spread * torch.randn((rows, k), generator=g)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)])
    return z.to(dev), t.to(dev), idx.to(dev)


def without_workspace(g, z, t, idx, lse, w, T):
    """frcnn_distill_bwd: rows that ops.distill_bwd splits with a workspace are walked instead."""
    from objectdetection_amd import _lib
    dts = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
    (rows, V), k = z.shape, t.shape[1]
    t, idx, g, lse = t.contiguous(), idx.contiguous(), g.contiguous(), lse.contiguous()
    grad = torch.empty((rows, V), dtype=z.dtype, device=z.device)
    assert _lib.lib.frcnn_distill_bwd(g.data_ptr(), z.data_ptr(), z.stride(0), dts[z.dtype], t.data_ptr(), dts[t.dtype], idx.data_ptr(),
                                      lse.data_ptr(), None if w is None else w.data_ptr(), rows, V, k, T, grad.data_ptr(), V,
                                      torch.cuda.current_stream().cuda_stream) == _lib.OK
    return grad


def check(got, ref, what):
    loss, grad, tol_l, tol_g = ref
    if "loss" in got:
        off = (got["loss"].double().cpu() - loss).abs()
        assert (off <= tol_l + 2.0 ** -23 * loss.abs()).all(), (what, "loss", float((off / tol_l).max()))
    g = got["d_logits"]
    off = (g.double().cpu() - grad).abs()
    tol = tol_g + torch.finfo(g.dtype).eps / 2 * grad.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 1e-37)
    assert (off <= tol).all(), (what, "gradient", float((off / tol).max()))


OFFSETS = [(1e4, 1.5, 2.0), (-3e5, 4.0, 20.0), (10.0, 1e-3, 2e-3), (0.0, 1e-18, 1e-18), (1e30, 1e18, 1e19)]


@pytest.mark.parametrize("rows,V,k", SHAPES)
@pytest.mark.parametrize("offset,T,spread", OFFSETS)
def test_the_teachers_logits_keep_their_differences(dev, rows, V, k, offset, T, spread):
    """The offset in the teacher's logits alone."""
    from objectdetection_amd import ops
    rows = min(rows, 40) if V > 5000 and rows < 200 else rows
    z, t, idx = make(V + k, dev, rows, V, k, spread)
    t = t + offset
    check(ops.distill_loss(z, t, idx, temperature=T), reference(z, t, idx, T), (offset, T))


@pytest.mark.parametrize("V,k", [(8, 5), (21, 8), (1203, 40), (4000, 100), (20003, 12), (70001, 70)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_entries_of_the_lowest_value_are_entries(dev, V, k, name):
    """A row of nothing else is uniform, beside others they weigh nothing; -inf alone is no entry.  At any temperature."""
    from objectdetection_amd import ops
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]
    for T in (0.25, 1.0, 3.0):
        z, t, idx = make(V, dev, 4, V, k, 2.0)
        t = t.to(dt)
        t[0] = torch.finfo(dt).min
        t[1, 1:] = torch.finfo(dt).min
        t[2, 1:] = -math.inf
        t[3] = torch.finfo(dt).max
        z, td = z.to(dt), t if k % 2 else t.float()
        got = ops.distill_loss(z, td, idx, temperature=T)
        check(got, reference(z, td, idx, T), T)
        assert (got["loss"][0] > 0) and got["loss"].isfinite().all()


@pytest.mark.parametrize("rows,V,k", SHAPES + [(1, 70001, 64), (1, 131072, 5), (700, 17000, 3), (2, 300001, 1024), (513, 70001, 2)])
@pytest.mark.parametrize("offset,T,spread", OFFSETS)
def test_the_backward_is_as_precise_as_the_fused_gradient(dev, rows, V, k, offset, T, spread):
    """The offset in the student's logits; both gradients are within the bounds, and each row of q sums to 1."""
    from objectdetection_amd import ops
    rows = min(rows, 40) if V > 5000 and rows < 200 else rows
    z, t, idx = make(V + k, dev, rows, V, k, spread)
    z = z + offset
    got = ops.distill_loss(z, t, idx, temperature=T)
    back = ops.distill_bwd(torch.ones(rows, device=dev), z, t, idx, got["lse"], temperature=T)
    some = torch.arange(0, rows, max(1, rows // 40))                # the reference of all would take minutes
    at = some.to(dev)
    ref = reference(z[at], t[at], idx[at], T)
    check({"loss": got["loss"][at], "d_logits": got["d_logits"][at]}, ref, (offset, T))
    walk = without_workspace(torch.ones(rows, device=dev), z, t, idx, got["lse"], None, T)
    for d in (back, walk):
        check({"d_logits": d[at]}, ref, (offset, T, "backward"))
        # sum_v (q_v - p_v) = 0: V roundings and the bounds above on either side
        assert (d.double().sum(1).abs() <= T * (2.0 ** -20 * 30 + 2 * (V / 256 + k + 32) * 2.0 ** -23 + V * 2.0 ** -126)).all()


@pytest.mark.parametrize("rows,V", [(1, 70001), (3, 40000), (2, 300001), (5, 131073)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("split", [True, False])
def test_backward_of_long_rows(dev, rows, V, name, split):
    """A row by one workgroup, by several, masked rows, rows without entries, -inf, NaN and +inf logits, strided rows, a captured
    call; rows alone give what they give among others."""
    from objectdetection_amd import ops
    bwd = ops.distill_bwd if split else without_workspace
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]
    z, t, idx = make(V, dev, 600, V, 70, 2.0) if rows == 3 else make(V, dev, 30, V, 70, 2.0)
    z, n = z.to(dt), z.shape[0]
    w = torch.ones(n, device=dev)
    idx[0, 3:9] = idx[0, :1]                       # a label listed often
    g = torch.linspace(-1.0, 2.0, n, device=dev)
    lse = torch.zeros(n, device=dev)
    every = bwd(g, z, t, idx, lse, w, 1.5)
    _, grad, _, tol = reference(z[:1], t[:1], idx[:1], 1.5)        # g[0] is -1
    off = (every[:1].double().cpu() + grad).abs()
    assert (off <= tol + torch.finfo(dt).eps / 2 * grad.abs() + (2.0 ** -25 if dt == torch.float16 else 1e-37)).all()
    for r in range(0, n - rows, max(1, n // 4)):
        s = slice(r, r + rows)
        assert torch.allclose(bwd(g[s], z[s], t[s], idx[s], lse[s], w[s], 1.5).float(), every[s].float(),
                              rtol=2 * torch.finfo(dt).eps, atol=2.0 ** -24)
    z, t, idx, g, lse, w = z[:6].clone(), t[:6], idx[:6].clone(), g[:6], lse[:6], w[:6].clone()
    w[0] = 0
    z[0] = math.nan
    idx[1] = -1
    z[2, 7] = math.nan
    z[3, 9] = math.inf
    z[4] = -math.inf
    z[5, ::2] = -math.inf
    got = bwd(g, z, t, idx, lse, w, 1.5)
    assert not got[:2].any()
    for r in (2, 3, 4):
        assert got[r].isnan().any()
    assert got[5].isfinite().all()
    wide = torch.zeros((6, V + 13), dtype=dt, device=dev)
    wide[:, 5:5 + V] = z
    same = lambda a, b: torch.equal(a.nan_to_num(nan=-77.0), b.nan_to_num(nan=-77.0))
    assert same(bwd(g, wide[:, 5:5 + V], t, idx, lse, w, 1.5), got)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        held = bwd(g, z, t, idx, lse, w, 1.5)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(held, got)


def test_the_backwards_workspace(dev):
    from objectdetection_amd import ops
    z, t, idx = make(1, dev, 3, 70001, 9, 2.0)
    one = torch.ones(3, device=dev)
    need = ops.distill_workspace_bytes(3, 70001, 9, torch.float32)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(ops.distill_bwd(one, z, t, idx, one, workspace=ws[:need]), ops.distill_bwd(one, z, t, idx, one))
    assert need > 0 and (ws[need:] == 255).all()
    with pytest.raises(ValueError):
        ops.distill_bwd(one, z, t, idx, one, workspace=ws[:need - 1])
    with pytest.raises(RuntimeError):
        ops.distill_bwd(one, z, t, idx, one, workspace=ws[4:need + 4])


def test_backward_of_rows_further_apart_than_32_bits(dev):
    from objectdetection_amd import ops
    for rows, V, ld in ((3, 70001, 1 << 31), (5, 40000, 1 << 30)):
        z, t, idx = make(rows, dev, rows, V, 5, 2.0)
        z = z.bfloat16()
        buf = torch.empty(((rows - 1) * ld + V,), dtype=torch.bfloat16, device=dev)
        far = torch.as_strided(buf, (rows, V), (ld, 1))
        far.copy_(z)
        g = torch.linspace(-1.0, 2.0, rows, device=dev)
        for bwd in (ops.distill_bwd, without_workspace):
            assert torch.equal(bwd(g, far, t, idx, g, None, 2.0), bwd(g, z, t, idx, g, None, 2.0))
        del buf, far
