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
