"""Distillation from a teacher's stored top logits (ops.distill_loss / ops.distill_bwd) against the
definition in float64.

Tolerances (derived before any run).  With A the largest |z/T|, |t/T| met plus ln V + ln k, every
logarithm is off by at most rel = 2^-22 A + (V / 256 + k + 32) 2^-23: a handful of float32 operations
on numbers up to A, and a float32 sum of V terms that 256 lanes or fewer share; a probability is
off by rel relative.  With D the largest |log p - log q| of the row's entries the loss
sum p (log p - log q) is off by (2 + D) rel, the gradient c (q - p) by |c| (q + p) rel, then each
stored value by one rounding of its type (float16: at least 2^-25).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(seed, dev, rows, V, k, dt, tdt=None, pad=False, scale=2.0):
    rng = np.random.default_rng(seed)
    z = torch.from_numpy((scale * rng.standard_normal((rows, V))).astype(np.float32)).to(dev).to(dt)
    t = torch.from_numpy((3 * rng.standard_normal((rows, k))).astype(np.float32)).to(dev).to(tdt or dt)
    idx = torch.from_numpy(np.stack([rng.permutation(V)[np.arange(k) % V] for _ in range(rows)])
                           if rows else np.zeros((0, k), np.int64)).to(dev)
    wt = None
    if pad:
        kept = torch.from_numpy(rng.integers(0, k + 1, (rows, 1))).to(dev)
        idx = torch.where(torch.arange(k, device=dev) < kept, idx, -1 - idx)
        wt = torch.from_numpy((rng.random(rows) * (rng.random(rows) > 0.25)).astype(np.float32)).to(dev)
    return z, t, idx, wt


def reference(z, t, idx, wt, T):
    """loss, lse, gradient of loss.sum() and the rows' rel, in float64 on the host, row by row."""
    z, t, idx = z.double().cpu() / T, t.double().cpu() / T, idx.cpu()
    rows, V = z.shape
    w = torch.ones(rows, dtype=torch.float64) if wt is None else wt.double().cpu()
    loss, lse, grad = torch.zeros(rows).double(), torch.zeros(rows).double(), torch.zeros_like(z)
    tol_l, tol_g = torch.zeros(rows).double(), torch.zeros_like(z)
    for r in range(rows):
        keep = (idx[r] >= 0) & (idx[r] < V) & (t[r] > -math.inf)
        if w[r] == 0 or not keep.any():
            continue
        i, tt = idx[r][keep], t[r][keep]
        log_p = torch.log_softmax(tt, 0)
        log_q = torch.log_softmax(z[r], 0)
        p, q = log_p.exp(), log_q.exp()
        loss[r] = w[r] * T * T * torch.where(p > 0, p * (log_p - log_q[i]), torch.zeros_like(p)).sum()
        lse[r] = torch.logsumexp(z[r], 0)
        full = torch.zeros(V).double().index_add_(0, i, p)
        grad[r] = w[r] * T * (q - full)
        fin = z[r][z[r].isfinite()]
        A = float(fin.abs().max()) + float(tt.abs().max()) + math.log(V) + math.log(idx.shape[1]) + 1
        rel = 2.0 ** -22 * A + (V / 256 + idx.shape[1] + 32) * 2.0 ** -23
        D = float((log_p - log_q[i]).abs().max())
        tol_l[r] = w[r].abs() * T * T * (2 + D) * rel
        tol_g[r] = (w[r] * T).abs() * (q + full) * rel
    return loss, lse, grad, tol_l, tol_g


def check(got, z, t, idx, wt, T, g=None):
    loss, lse, grad, tol_l, tol_g = reference(z, t, idx, wt, T)
    if "loss" in got:
        assert ((got["loss"].double().cpu() - loss).abs() <= tol_l + 2.0 ** -23 * loss.abs()).all()
        assert ((got["lse"].double().cpu() - lse).abs() <= tol_l / T ** 2 / 2 + 2.0 ** -21 * (1 + lse.abs())).all()
    if got["d_logits"] is not None:
        if g is not None:
            grad, tol_g = grad * g[:, None], tol_g * g.abs()[:, None]
        d = got["d_logits"]
        assert d.dtype == z.dtype and d.shape == z.shape
        off = (d.double().cpu() - grad).abs()
        tol = tol_g * 1.01 + torch.finfo(z.dtype).eps / 2 * grad.abs() + (2.0 ** -25 if z.dtype == torch.float16 else 1e-37)
        assert (off <= tol).all(), float((off / tol).max())


SIZES = [(1, 1, 1), (5, 2, 2), (7, 21, 8), (300, 21, 21), (3, 64, 3), (9, 65, 5), (4, 257, 33), (2, 1031, 100),
         (33, 4096, 64), (700, 100, 12), (260, 700, 40), (3, 20011, 17), (1, 131072, 64), (2, 66000, 1), (5, 40, 40), (2, 2500, 1024)]


@pytest.mark.parametrize("rows,V,k", SIZES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_loss_and_gradients(dev, rows, V, k, name):
    from objectdetection_amd import ops
    dt = TYPES[name]
    for T, pad, tdt in ((1.0, False, None), (2.5, True, torch.float32), (0.7, True, None)):
        z, t, idx, wt = make(rows + V + k, dev, rows, V, k, dt, tdt, pad)
        got = ops.distill_loss(z, t, idx, weight=wt, temperature=T)
        check(got, z, t, idx, wt, T)
        fwd = ops.distill_loss(z, t, idx, weight=wt, temperature=T, want_grad=False)
        assert fwd["d_logits"] is None and torch.equal(fwd["loss"], got["loss"]) and torch.equal(fwd["lse"], got["lse"])
        g = torch.linspace(-1.5, 2.0, rows, device=dev)
        d = ops.distill_bwd(g, z, t, idx, got["lse"], weight=wt, temperature=T)
        check({"d_logits": d}, z, t, idx, wt, T, g.double().cpu())


def test_grad_scale_strided_logits_and_leading_dimensions(dev):
    from objectdetection_amd import ops
    z, t, idx, _ = make(1, dev, 12, 50, 4, torch.float32)
    wide = torch.zeros((12, 83), device=dev)
    wide[:, 5:55] = z
    a = ops.distill_loss(z, t, idx, temperature=2.0, grad_scale=0.125)
    b = ops.distill_loss(wide[:, 5:55], t, idx, temperature=2.0, grad_scale=0.125)
    c = ops.distill_loss(z.view(3, 4, 50), t.view(3, 4, 4), idx.view(3, 4, 4), temperature=2.0, grad_scale=0.125)
    assert c["loss"].shape == (3, 4) and c["d_logits"].shape == (3, 4, 50)
    for k in a:
        assert torch.equal(a[k], b[k]) and torch.equal(a[k].reshape(-1), c[k].reshape(-1))
    check(dict(loss=a["loss"], lse=a["lse"], d_logits=a["d_logits"] * 8), z, t, idx, None, 2.0)


@pytest.mark.parametrize("V,k", [(21, 5), (64, 64), (300, 7), (5000, 70), (21, 100), (70000, 300)])
def test_label_listed_twice_counts_twice(dev, V, k):
    from objectdetection_amd import ops
    z, t, idx, _ = make(3, dev, 6, V, k, torch.float32)
    idx[:, 1:4] = idx[:, :1]
    idx[3] = V - 1
    check(ops.distill_loss(z, t, idx, temperature=1.5), z, t, idx, None, 1.5)


@pytest.mark.parametrize("V", [21, 300, 9001, 40000])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_masked_rows_infinities_and_nan(dev, V, name):
    """Rows that take no part are not read (NaN there changes nothing) and get zeros; -inf logits of
    teacher and student; the lowest finite value as a mask; NaN and +inf reach their own row only."""
    from objectdetection_amd import ops
    inf, nan, dt = math.inf, math.nan, TYPES[name]
    z, t, idx, _ = make(5, dev, 12, V, 5, dt)
    wt = torch.ones(12, device=dev)
    z[0] = nan
    wt[0] = 0                                  # masked: nothing of it is read
    t[0] = nan
    idx[1] = -1
    z[1] = nan                                 # no entry
    t[2] = -inf                                # no entry either
    t[3, 1:] = -inf                            # one entry
    idx[4, 2:] = V + 7                         # labels outside
    t[4, 2:] = nan
    low = torch.finfo(dt).min
    z[5, (idx[5, 0] + 1) % V] = -inf           # a masked student label, not the teacher's (or maybe)
    z[6, idx[6, 0]] = -inf                     # the teacher's own label masked: an infinite loss
    z[7] = torch.where(torch.arange(V, device=dev) % 2 == 0, z[7], torch.full_like(z[7], low))
    z[8, 1] = nan
    z[9, 1] = inf
    t[10, 0] = nan
    z[11] = -inf
    got = ops.distill_loss(z, t, idx, weight=wt)
    loss, lse, d = got["loss"].cpu(), got["lse"].cpu(), got["d_logits"].float().cpu()
    for r in (0, 1, 2):
        assert loss[r] == 0 and lse[r] == 0 and not d[r].any()
    assert loss[6] == inf and d[6].isfinite().all()
    for r in (8, 9, 10, 11):
        assert loss[r].isnan() and d[r].isnan().any()
    keep = [3, 4]
    check({k: v[keep] for k, v in got.items()}, z[keep], t[keep], idx[keep], None, 1.0)
    # the gradient of the rows with an infinite or huge loss is finite all the same
    _, _, g, _, tol = reference(z[6:7], t[6:7], idx[6:7], None, 1.0)
    assert ((d[6:7] - g).abs() <= tol + torch.finfo(dt).eps * g.abs() + 2.0 ** -25).all()
    g5 = reference(z[5:6], t[5:6], idx[5:6], None, 1.0)[2]
    assert ((d[5:6] - g5).abs() <= 1e-4 + torch.finfo(dt).eps * g5.abs()).all()
    assert d[7].isfinite().all()
    back = ops.distill_bwd(torch.ones(12, device=dev), z, t, idx, got["lse"], weight=wt)
    for r in (0, 1, 2):
        assert not back[r].any()
    assert torch.allclose(back[3:5].float(), got["d_logits"][3:5].float(), atol=1e-5, rtol=2 ** -6)


def test_huge_logits_do_not_overflow(dev):
    from objectdetection_amd import ops
    for dt, big in ((torch.float32, 1e30), (torch.float16, 6e4), (torch.bfloat16, 1e30)):
        z = torch.tensor([[big, 0.0, -big], [big, big, -big]], device=dev).to(dt)
        t = torch.tensor([[big, 0.0], [1.0, 1.0]], device=dev).to(dt)
        got = ops.distill_loss(z, t, torch.tensor([[0, 1], [0, 1]], device=dev))
        assert got["loss"].tolist() == [0.0, 0.0]
        assert got["d_logits"].float().abs().max() <= 1e-6


def test_no_rows_and_same_bits(dev):
    from objectdetection_amd import ops
    z, t, idx, _ = make(1, dev, 0, 50, 4, torch.float32)
    got = ops.distill_loss(z, t, idx)
    assert got["loss"].shape == (0,) and got["d_logits"].shape == (0, 50)
    for V in (21, 700, 50000):
        z, t, idx, wt = make(1, dev, 9, V, 6, torch.bfloat16, pad=True)
        a = ops.distill_loss(z, t, idx, weight=wt)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                b = ops.distill_loss(z, t, idx, weight=wt)
                assert all(torch.equal(a[k], b[k]) for k in a)
        torch.cuda.current_stream().wait_stream(side)


def test_captured_call_replays(dev):
    from objectdetection_amd import ops
    for V in (21, 40000):
        z, t, idx, wt = make(1, dev, 9, V, 6, torch.bfloat16, pad=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a = ops.distill_loss(z, t, idx, weight=wt)
            d = ops.distill_bwd(a["loss"], z, t, idx, a["lse"], weight=wt)
        for step in range(4):
            z.copy_(torch.randn_like(z))
            graph.replay()
            torch.cuda.synchronize()
            b = ops.distill_loss(z, t, idx, weight=wt)
            assert all(torch.equal(a[k], b[k]) for k in a), step
            assert torch.equal(d, ops.distill_bwd(b["loss"], z, t, idx, b["lse"], weight=wt)), step


def test_gradient_against_differences(dev):
    from objectdetection_amd import ops
    z, t, idx, _ = make(4, dev, 2, 30, 5, torch.float32)
    got = ops.distill_loss(z, t, idx, temperature=1.5)["d_logits"].double().cpu()
    num, h = torch.zeros(2, 30).double(), 1e-5
    for r in range(2):
        for v in range(30):
            f = []
            for s in (h, -h):
                y = z.double()
                y[r, v] += s
                f.append(float(reference(y, t, idx, None, 1.5)[0].sum()))
            num[r, v] = (f[0] - f[1]) / (2 * h)
    assert (got - num).abs().max() <= 1e-5


def test_refusals(dev):
    from objectdetection_amd import ops
    z, t, idx, wt = make(1, dev, 4, 20, 3, torch.float32, pad=True)
    one = torch.ones(4, device=dev)
    for bad, err in (
            (lambda: ops.distill_loss(z.double(), t, idx), TypeError),
            (lambda: ops.distill_loss(z, t.half(), idx), TypeError),
            (lambda: ops.distill_loss(z, t, idx.int()), TypeError),
            (lambda: ops.distill_loss(z, t[:3], idx[:3]), ValueError),
            (lambda: ops.distill_loss(z, t, idx[:, :2]), ValueError),
            (lambda: ops.distill_loss(z, t, idx, weight=wt[:2]), ValueError),
            (lambda: ops.distill_loss(z, t, idx, weight=wt.half()), TypeError),
            (lambda: ops.distill_loss(z, t, idx, temperature=0.0), ValueError),
            (lambda: ops.distill_loss(z, t, idx, temperature=math.nan), ValueError),
            (lambda: ops.distill_loss(z, t, idx, temperature=math.inf), ValueError),
            (lambda: ops.distill_loss(z, t, idx, temperature=1e-19), ValueError),
            (lambda: ops.distill_loss(z.cpu(), t, idx), RuntimeError),
            (lambda: ops.distill_loss(z, t.cpu(), idx), RuntimeError),
            (lambda: ops.distill_loss(z, t, idx.cpu()), RuntimeError),
            (lambda: ops.distill_bwd(one[:3], z, t, idx, one), ValueError),
            (lambda: ops.distill_bwd(one, z, t, idx, one.double()), TypeError),
            (lambda: ops.distill_loss(z, t.repeat(1, 400), idx.repeat(1, 400)), RuntimeError)):
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("name,rows,V", [("bf16", 210, 40000), ("f32", 210, 20003), ("f16", 70, 131072), ("f32", 70, 65000)])
def test_many_long_rows(dev, name, rows, V):
    """Rows of up to 16,384 pieces of 16 bytes stay in one workgroup when there are many."""
    from objectdetection_amd import ops
    assert ops.distill_workspace_bytes(rows, V, 9, TYPES[name]) == 0
    z, t, idx, wt = make(rows + V, dev, rows, V, 9, TYPES[name], torch.float32, True)
    check(ops.distill_loss(z, t, idx, weight=wt, temperature=1.5), z, t, idx, wt, 1.5)


def test_rows_further_apart_than_32_bits(dev):
    from objectdetection_amd import ops
    for rows, V, ld in ((40, 21, 1 << 27), (40, 5003, 1 << 27), (3, 70001, 1 << 31)):
        z, t, idx, wt = make(rows, dev, rows, V, 5, torch.bfloat16, torch.float32, True)
        buf = torch.empty(((rows - 1) * ld + V,), dtype=torch.bfloat16, device=dev)
        far = torch.as_strided(buf, (rows, V), (ld, 1))
        far.copy_(z)
        a, b = (ops.distill_loss(q, t, idx, weight=wt, temperature=2.0) for q in (far, z))
        assert all(torch.equal(a[k], b[k]) for k in a)
        g = torch.ones(rows, device=dev)
        assert torch.equal(ops.distill_bwd(g, far, t, idx, a["lse"], wt, 2.0), ops.distill_bwd(g, z, t, idx, a["lse"], wt, 2.0))
        del buf, far


@pytest.mark.parametrize("V,k,labels", [(5000, 65, 30), (5000, 1024, 1), (5000, 1024, 5), (70000, 1024, 400), (300, 700, 300),
                                        (1000, 130, 129), (40000, 1024, 1024), (3, 193, 3), (1024, 192, 150), (1024, 193, 190)])
def test_many_entries_with_the_same_labels(dev, V, k, labels):
    """More than 64 entries: every label in the list once, a few times, or in all of it; the same bits each time."""
    rng = np.random.default_rng(V + k + labels)
    z, t, _, _ = make(V, dev, 5, V, k, torch.float32)
    of = np.stack([rng.permutation(V)[:labels] for _ in range(5)])
    idx = np.take_along_axis(of, rng.integers(0, labels, (5, k)) if labels < k else np.tile(rng.permutation(k), (5, 1)), 1)
    idx[1, ::3] = -1
    idx[2, 1:] = V
    idx[3, :] = idx[3, 0]
    idx[4, :] = -1 if k % 2 else V + 7
    idx = torch.from_numpy(idx).to(dev)
    from objectdetection_amd import ops
    got = ops.distill_loss(z, t, idx, temperature=1.5)
    check(got, z, t, idx, None, 1.5)
    g = torch.ones(5, device=dev)
    d = ops.distill_bwd(g, z, t, idx, got["lse"], None, 1.5)
    check({"d_logits": d}, z, t, idx, None, 1.5)
    for _ in range(3):
        assert torch.equal(ops.distill_loss(z, t, idx, temperature=1.5)["d_logits"], got["d_logits"])
        assert torch.equal(ops.distill_bwd(g, z, t, idx, got["lse"], None, 1.5), d)


@pytest.mark.parametrize("rows,V,k", [(9, 3, 40), (6, 1, 17), (70, 17, 17), (33, 21, 40), (5, 129, 64), (65, 511, 63), (3, 2049, 64),
                                      (7, 4096, 20), (5, 1024, 1), (40, 92, 33), (3, 2048, 2), (17, 8, 31)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_short_rows(dev, rows, V, k, name):
    """Several rows per wave: row ends inside a piece, entries that do not fill their lanes, labels listed twice."""
    from objectdetection_amd import ops
    dt = TYPES[name]
    for pad, tdt in ((False, None), (True, torch.float32)):
        z, t, idx, wt = make(rows * V + k, dev, rows, V, k, dt, tdt, pad)
        idx[:, k // 2:] = torch.where(idx[:, k // 2:] >= 0, idx[:, :k - k // 2], idx[:, k // 2:])
        got = ops.distill_loss(z, t, idx, weight=wt, temperature=1.5)
        check(got, z, t, idx, wt, 1.5)
        g = torch.linspace(-1.5, 2.0, rows, device=dev)
        check({"d_logits": ops.distill_bwd(g, z, t, idx, got["lse"], wt, 1.5)}, z, t, idx, wt, 1.5, g.double().cpu())


def test_short_rows_write_nothing_behind_their_end(dev):
    """A strided gradient: what lies between the rows keeps its bytes (the C entry takes the stride)."""
    from objectdetection_amd import _lib
    for V, k, ldg in ((21, 8, 24), (91, 8, 100), (9, 20, 9), (5, 20, 7), (1203, 32, 1210)):
        z, t, idx, _ = make(V, dev, 37, V, k, torch.bfloat16, torch.float32)
        buf = torch.full((37 * ldg + 64,), 7.0, dtype=torch.bfloat16, device=dev)
        loss, lse = torch.empty(37, device=dev), torch.empty(37, device=dev)
        s = torch.cuda.current_stream().cuda_stream
        assert _lib.lib.frcnn_distill_loss(z.data_ptr(), V, _lib.DT_BF16, t.data_ptr(), _lib.DT_F32, idx.data_ptr(), None, 37, V, k, 2.0,
                                           1.0, loss.data_ptr(), lse.data_ptr(), buf.data_ptr(), ldg, None, 0, s) == _lib.OK
        rows = buf[:37 * ldg].view(37, ldg)
        check(dict(loss=loss, lse=lse, d_logits=rows[:, :V]), z, t, idx, None, 2.0)
        assert (rows[:, V:] == 7).all() and (buf[37 * ldg:] == 7).all()
