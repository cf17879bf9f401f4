"""The precision in which dz = d_out * act'(pre) enters the products of ops.dense_bwd: where it is no value of
the layer's type (GELU, SiLU, a float32 d_out) it is the sum of two.

Derived before any run:
  pair       dz is held within u |dz|: each of the two roundings leaves eps / 2 of what it rounds, so u = (eps / 2)^2,
             2^-16 in bfloat16 and 2^-22 in float16;
  gradients  against float64 in the 2-norm: the stored values are rounded once, by r = |round(ref) - ref|, and only
             the pair and float32 sums (together below 2^-15 of the result, r is 2^-10 or more of it in bfloat16 and
             2^-13 in float16) come on top: at most 1.02 r in float16, 1.02 r in bfloat16.  A dz rounded to the
             type adds an error of r's size that is independent of it: 1.4 r;
  two terms  where the reduction has few terms the bound holds value by value: the terms' u |dz| |w|, act' within
             2e-6 (1 + |z|) (float32 exp2, rcp and the polynomial's 1.3e-6, slopes up to 1.13), one rounding of the result.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().to("cpu").double()


def grad64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def make(seed, dev, M, K, N, dt, layout, d_dt):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    x, w = n(M, K).to(dev).to(dt), n(K, N) / K ** 0.5
    w = w.to(dev).to(dt) if layout == "kn" else w.t().contiguous().to(dev).to(dt).t()
    return x, w, n(M, N).to(dev).to(d_dt), n(M, N).to(dev).to(dt)


# few rows (by themselves and by tiles), both products in one launch, every tile size, split reductions, odd rows
SIZES = [(1, 64, 48), (7, 333, 100), (20, 4104, 72), (32, 4104, 2056), (40, 40, 40), (300, 203, 85), (1111, 779, 333),
         (130, 8200, 84), (2000, 1024, 1000), (4097, 264, 2051), (3900, 2056, 264), (900, 33, 5000)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("name,act,wide", [("f16", "silu", False), ("bf16", "gelu", False), ("f16", "none", True),
                                           ("bf16", "relu", True), ("f16", "gelu", True)])
def test_gradients_are_rounded_once(dev, M, K, N, layout, name, act, wide):
    from objectdetection_amd import ops
    dt = TYPES[name]
    x, w, d, pre = make(M + N, dev, M, K, N, dt, layout, torch.float32 if wide else dt)
    g = ops.dense_bwd(d, x, w, None if act == "none" else pre, act)
    dz = f64(d) * grad64(f64(pre), act)
    for key, ref in (("d_x", dz @ f64(w).t()), ("d_weight", f64(x).t() @ dz), ("d_bias", dz.sum(0))):
        if ref.numel() < 500:
            continue                           # too few values for their mean rounding to be the expected one
        once = float((ref.to(dt).double() - ref).norm())
        assert float((f64(g[key]) - ref).norm()) <= 1.02 * once, key


@pytest.mark.parametrize("M,K,N", [(24, 64, 100), (70, 40, 333), (1030, 136, 84), (2100, 2056, 2064)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_few_terms_value_by_value(dev, M, K, N, layout, name):
    """Two values of d_out in a row (so d_x has two terms) and one row of x for a column of d_weight."""
    from objectdetection_amd import ops
    dt = TYPES[name]
    x, w, d, pre = make(M, dev, M, K, N, dt, layout, dt)
    row = torch.arange(M, device=dev)
    keep = torch.zeros((M, N), dtype=torch.bool, device=dev)
    keep[row, row % N] = True
    keep[row, (7 * row + 3) % N] = True
    d = torch.where(keep, d, torch.zeros_like(d))
    wide = torch.where(keep, torch.randn((M, N), device=dev), torch.zeros((M, N), device=dev))
    u = (torch.finfo(dt).eps / 2) ** 2
    for act, up in (("silu", d), ("gelu", d), ("none", wide)):
        g = ops.dense_bwd(up, x, w, None if act == "none" else pre, act)
        z, D = f64(pre), f64(up)
        dz = D * grad64(z, act)
        err = u * dz.abs() + (0 if act == "none" else 2e-6 * (1 + z.abs()) * D.abs()) + 2.0 ** -34
        for key, ref, tol in (("d_x", dz @ f64(w).t(), err @ f64(w).abs().t() + 2.0 ** -22 * (dz.abs() @ f64(w).abs().t())),
                              ("d_weight", f64(x).t() @ dz, f64(x).abs().t() @ err + (1 + M / N) * 2.0 ** -21 * (f64(x).abs().t() @ dz.abs()))):
            off = (f64(g[key]) - ref).abs()
            tol = 1.01 * tol + torch.finfo(dt).eps / 2 * ref.abs() + (2.0 ** -25 if dt == torch.float16 else 1e-37)
            assert (off <= tol).all(), (act, key, float((off / tol).max()))


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_cancelling_terms_of_a_float32_gradient(dev, name):
    """Rows that differ by less than a step of the 16-bit type: what is left of them is the difference."""
    from objectdetection_amd import ops
    dt = TYPES[name]
    for M, K, N in ((2, 24, 16), (64, 24, 40), (512, 520, 264)):
        d = torch.ones((M, N), device=dev)
        d[1::2] = -1.0 - torch.finfo(dt).eps / 4 * torch.arange(1, N + 1, device=dev) / N
        x = torch.ones((M, K), device=dev).to(dt)
        w = torch.ones((K, N), device=dev).to(dt)
        g = ops.dense_bwd(d, x, w)
        want = f64(d).sum(0)[None].expand(K, N)            # M / 2 times -eps / 4 times n / N
        # the pair leaves (eps / 2)^2 of every 1, float32 sums of M of them M 2^-24: of a difference of M eps / 8 and more
        tol = M * (torch.finfo(dt).eps / 2) ** 2 + M * M * 2.0 ** -24 + torch.finfo(dt).eps / 2 * want.abs()
        assert ((f64(g["d_weight"]) - want).abs() <= tol).all()
        assert float(f64(g["d_weight"]).abs().min()) > 0 or M == 2


def test_infinities_and_nan_reach_their_own_rows(dev):
    from objectdetection_amd import ops
    for dt in TYPES.values():
        for M, K, N in ((20, 40, 24), (130, 72, 100)):
            x, w, d, pre = make(3, dev, M, K, N, dt, "kn", dt)
            d[3, 5], d[7, 1] = math.inf, math.nan
            g = ops.dense_bwd(d, x, w, pre, "silu")
            bad = ~g["d_x"].isfinite().all(1)
            assert bad.nonzero().flatten().tolist() == [3, 7] and not g["d_x"][[3, 7]].isfinite().any()
            assert (~g["d_weight"].isfinite().all(0)).nonzero().flatten().tolist() == [1, 5]
            assert g["d_bias"].isnan().nonzero().flatten().tolist() == [1]


@pytest.mark.parametrize("power", [-30, -20, -14, 12, 20])
@pytest.mark.parametrize("M,K,N", [(20, 264, 100), (300, 203, 85), (2000, 1024, 264), (4097, 264, 2051)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_float32_gradients_outside_the_range_of_float16(dev, power, M, K, N, act):
    """The gradients are in range (W and x make up for it as far as they can), d_out is not; infinities and zeros
    in it do not move its scale."""
    from objectdetection_amd import ops
    x, w, d, pre = make(power + M, dev, M, K, N, torch.float16, "nk", torch.float32)
    f = 2.0 ** max(-13, min(-power, 13))
    x, w, d = (x.float() * f).half(), (w.float() * f).half(), d * 2.0 ** power
    d[:, 1] = 0
    g = ops.dense_bwd(d, x, w, None if act == "none" else pre, act)
    dz = f64(d) * grad64(f64(pre), act)
    for key, ref in (("d_x", dz @ f64(w).t()), ("d_weight", f64(x).t() @ dz)):
        assert float(ref.abs().max()) < 60000
        once = float((ref.half().double() - ref).norm())
        assert float((f64(g[key]) - ref).norm()) <= 1.02 * once, key
    d[3, 7] = math.inf
    h = ops.dense_bwd(d, x, w, None if act == "none" else pre, act)
    keep = torch.arange(M, device=dev) != 3
    assert torch.equal(h["d_x"][keep], g["d_x"][keep]) and not h["d_x"][3].isfinite().any()
    keep = torch.arange(N, device=dev) != 7
    assert torch.equal(h["d_weight"][:, keep], g["d_weight"][:, keep])


def test_a_scaled_gradient_gives_scaled_gradients(dev):
    """A power of two in a float32 d_out is one in the results: the same bits, from float32's smallest values on."""
    from objectdetection_amd import ops
    x, w, d, _ = make(9, dev, 70, 96, 40, torch.float16, "kn", torch.float32)
    ref = ops.dense_bwd(d, x, w)
    for power in (-9, -5, 3):
        g = ops.dense_bwd(d * 2.0 ** power, x, w)
        for key in ("d_x", "d_weight"):
            normal = ref[key].abs() >= 2.0 ** (-14 - min(power, 0))
            assert torch.equal(g[key][normal].float(), ref[key][normal].float() * 2.0 ** power)
    for up in (torch.zeros_like(d), torch.full_like(d, 2.0 ** -149)):
        g = ops.dense_bwd(up, x, w)
        assert not g["d_x"].any() and not g["d_weight"].any()
    only = torch.full_like(d, math.nan)
    assert ops.dense_bwd(only, x, w)["d_x"].isnan().all()


@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_weight_gradients_lie_as_the_weights_do(dev, layout):
    from objectdetection_amd import ops
    for M, K, N in ((5, 24, 40), (300, 96, 85)):
        x, w, d, pre = make(1, dev, M, K, N, torch.bfloat16, layout, torch.bfloat16)
        for act in ("none", "gelu"):
            g = ops.dense_bwd(d, x, w, pre, act)["d_weight"]
            assert g.shape == w.shape and g.stride() == w.stride()


def test_a_strided_float32_gradient_and_a_dirty_workspace(dev):
    """Between the rows of d_out, and in the workspace before the call, stand NaN and infinities."""
    from objectdetection_amd import ops
    for M, K, N in ((20, 264, 21), (300, 203, 85), (5000, 40, 84)):
        x, w, d, pre = make(M, dev, M, K, N, torch.float16, "nk", torch.float32)
        d = d * 1e-7
        wide = torch.full((M, N + 11), math.inf, device=dev)
        wide[:, 4] = math.nan
        wide[:, 5:5 + N] = d
        for act in ("none", "silu"):
            z = None if act == "none" else pre
            need = ops.dense_bwd_workspace_bytes(M, K, N, 1)
            ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)
            g, h = ops.dense_bwd(d, x, w, z, act), ops.dense_bwd(wide[:, 5:5 + N], x, w, z, act, workspace=ws[:need])
            assert all(torch.equal(g[k], h[k]) for k in g) and (ws[need:] == 255).all() and g["d_x"].any()


def test_captured_with_the_scale_of_each_replay(dev):
    """A float16 layer's float32 gradient of another size in every replay; two graphs with a workspace each."""
    from objectdetection_amd import ops
    for M, K, N in ((700, 4096, 84), (24, 520, 21), (1111, 779, 333)):
        x, w, d, pre = make(M, dev, M, K, N, torch.float16, "kn", torch.float32)
        side, graphs = torch.cuda.Stream(), []
        for _ in range(2):
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                graphs.append((graph, ops.dense_bwd(d, x, w, pre, "silu")))
        for f in (1.0, 1e-9, 3e5, 1e-4):
            d.copy_(f * torch.randn_like(d))
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            want = ops.dense_bwd(d, x, w, pre, "silu")
            assert all(torch.equal(got[k], want[k]) for _, got in graphs for k in want), f


def test_parts_of_dz_beyond_4_gib(dev):
    """600,000 rows of 4,096: each part of dz takes 4.9 GB."""
    from objectdetection_amd import ops
    M, K, N = 600_000, 8, 4096
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((M, K), generator=g, device=dev).bfloat16()
    w = torch.randn((K, N), generator=g, device=dev).bfloat16()
    d = torch.randn((M, N), generator=g, device=dev, dtype=torch.bfloat16)
    pre = torch.randn((M, N), generator=g, device=dev, dtype=torch.bfloat16)
    got = ops.dense_bwd(d, x, w, pre, "silu")
    dw, db = torch.zeros((K, N), dtype=torch.float64, device=dev), torch.zeros(N, dtype=torch.float64, device=dev)
    for r in range(0, M, 50_000):
        s = slice(r, r + 50_000)
        z = pre[s].double()
        q = torch.sigmoid(z)
        dz = d[s].double() * q * (1 + z * (1 - q))
        dw += x[s].double().t().contiguous() @ dz
        db += dz.sum(0)
        ref = dz[-3000:] @ w.double().t().contiguous()
        once = float((ref.bfloat16().double() - ref).norm())
        assert float((got["d_x"][r + 47_000:r + 50_000].double() - ref).norm()) <= 1.02 * once
    # float32 sums of 600,000 terms: relative to the sums of their sizes 2^-24 a step of 32 and a slice, sqrt of their number
    for key, ref in (("d_weight", dw), ("d_bias", db)):
        once = float((ref.bfloat16().double() - ref).norm())
        assert float((got[key].double() - ref).norm()) <= 1.02 * once + 2.0 ** -24 * math.sqrt(M / 32) * math.sqrt(M) * math.sqrt(ref.numel()), key
