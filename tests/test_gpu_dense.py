"""The head's dense layer on 16-bit inputs (ops.dense_fwd / ops.dense_bwd) against the same formulas
in float64, element by element.

Tolerances are first-order rounding bounds, derived before any run:
  sums     a float32 sum of n products in any order is off by at most n * 2^-23 * sum|x w| (products of
           16-bit values are exact; 2^-23 also covers additions that truncate);
  GELU     Phi is within 2e-6 relative (1.3e-6 polynomial, exp2 and rcp 1 ulp each), SiLU's sigmoid
           within 1e-6; both activations have slopes of at most 1.13, their derivatives are
           within 1e-5 * |d_out| absolute;
  output   one rounding to nearest: eps / 2 * |value|, at least half a step of float16's subnormals
           (2^-25); bfloat16 has float32's exponent range;
  dz       is rounded once more before the two products (GELU and SiLU only; the others' dz is
           d_out or 0): eps / 2 * |dz| through the absolute operand.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(rng, dev, M, K, N, dt, layout="kn", bias=True, residual=False):
    t = lambda a: torch.from_numpy(a.astype(np.float32)).to(dev).to(dt)
    x = t(np.maximum(rng.standard_normal((M, K)), -0.3))
    w = rng.standard_normal((K, N)) / math.sqrt(K)
    w = t(w) if layout == "kn" else t(np.ascontiguousarray(w.T)).t()
    return (x, w, t(rng.standard_normal(N)) if bias else None,
            t(rng.standard_normal((M, N))) if residual else None)


def f64(t):
    return None if t is None else t.detach().to("cpu").double()


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def grad64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def within(got, ref, tol, what):
    got = f64(got)
    assert got.shape == ref.shape, what
    off = (got - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by " \
        f"{float((off / tol).nan_to_num(nan=9e9).max()):.3g} times its tolerance"


def rounding(v, dt):
    return torch.finfo(dt).eps / 2 * v.abs() * 1.001 + (2.0 ** -25 if dt == torch.float16 else 1e-37)


def check_fwd(x, w, b, res, act, out, pre=None, odt=None):
    X, W, K = f64(x.reshape(-1, w.shape[0])), f64(w), w.shape[0]
    z = X @ W + (0 if b is None else f64(b))
    err = K * 2.0 ** -23 * (X.abs() @ W.abs() + (0 if b is None else f64(b).abs())) + 2.0 ** -23 * z.abs()
    dt = x.dtype
    if pre is not None:
        within(pre.reshape(z.shape), z, err + rounding(z, dt), "pre")
    ref = act64(z, act)
    err = 1.13 * err + 4e-6 * z.abs()
    if res is not None:
        r = f64(res).reshape(z.shape)
        ref = ref + r
        err = err + 2.0 ** -23 * (ref.abs() + r.abs())
    within(out.reshape(z.shape), ref, err + (rounding(ref, dt) if odt is None else 2.0 ** -23 * ref.abs()), "out")


def check_bwd(x, w, d, pre, act, g):
    X, W, D = f64(x.reshape(-1, w.shape[0])), f64(w), f64(d.reshape(-1, w.shape[1]))
    M, N, dt = X.shape[0], W.shape[1], x.dtype
    dz = D * (1 if act == "none" else grad64(f64(pre).reshape(D.shape), act))
    edz = 1e-5 * D.abs() if act in ("gelu", "silu") else torch.zeros_like(D)
    erd = edz + (rounding(dz, dt) if act in ("gelu", "silu") or d.dtype != dt else 0)
    if g["d_x"] is not None:
        ref = dz @ W.t()
        tol = erd @ W.abs().t() + N * 2.0 ** -23 * (dz.abs() + erd) @ W.abs().t() + rounding(ref, dt)
        within(g["d_x"].reshape(M, -1), ref, tol * 1.01, "d_x")
    if g["d_weight"] is not None:
        ref = X.t() @ dz
        tol = X.abs().t() @ erd + M * 2.0 ** -23 * X.abs().t() @ (dz.abs() + erd) + rounding(ref, dt)
        within(g["d_weight"], ref, tol * 1.01, "d_weight")
    if g["d_bias"] is not None:
        ref = dz.sum(0)
        tol = edz.sum(0) + M * 2.0 ** -23 * dz.abs().sum(0) + rounding(ref, dt)
        within(g["d_bias"], ref, tol * 1.01, "d_bias")


SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (17, 64, 16), (1, 4096, 520), (16, 1536, 256), (33, 96, 21),
         (130, 200, 84), (257, 1003, 331), (128, 128, 128), (300, 72, 1032), (1030, 264, 136), (2, 7, 2050), (32, 1000, 100), (31, 9001, 40),
         (5, 25088, 24), (1, 8200, 33), (33, 4104, 48)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_forward_sizes_and_layouts(dev, M, K, N, layout):
    from objectdetection_amd import ops
    for n, (name, act) in enumerate((("bf16", "relu"), ("f16", "gelu"), ("bf16", "none"), ("f16", "silu"))):
        x, w, b, res = make(np.random.default_rng(M + K + N + n), dev, M, K, N, TYPES[name], layout, n != 2, n > 0)
        out, pre = ops.dense_fwd(x, w, b, act=act, residual=res, want_pre=True)
        assert out.dtype == x.dtype and pre.dtype == x.dtype
        check_fwd(x, w, b, res, act, out, pre)


@pytest.mark.parametrize("M,K,N", SIZES + [(5001, 40, 24), (2048, 16, 84)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_backward_sizes_and_layouts(dev, M, K, N, layout):
    from objectdetection_amd import ops
    for n, (name, act) in enumerate((("bf16", "none"), ("f16", "gelu"), ("bf16", "relu"), ("f16", "silu"))):
        rng = np.random.default_rng(M + 2 * K + N + n)
        x, w, b, d = make(rng, dev, M, K, N, TYPES[name], layout, True, True)
        pre = ops.dense_fwd(x, w, b, want_pre=True)[1]
        g = ops.dense_bwd(d, x, w, pre=pre, act=act)
        assert g["d_weight"].stride() == w.contiguous().stride() if layout == "kn" else True
        check_bwd(x, w, d, pre, act, g)


@pytest.mark.parametrize("M,K,N", [(4100, 200, 2056), (2304, 96, 3000), (2049, 64, 2880), (4097, 33, 2051), (3900, 32, 4104)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_large_tiles(dev, M, K, N, layout):
    """Enough output for the largest workgroup tiles, ragged at their edges, short and odd in k: the
    forward, and as d_weight's and d_x's sizes the backward."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(M + K)
    x, w, b, res = make(rng, dev, M, K, N, torch.bfloat16, layout, True, True)
    out, pre = ops.dense_fwd(x, w, b, act="silu", residual=res, want_pre=True)
    check_fwd(x, w, b, res, "silu", out, pre)
    xt, wt, _, d = make(rng, dev, K, M, N, torch.float16, layout, False, True)       # d_weight [M,N]
    check_bwd(xt, wt, d, None, "none", ops.dense_bwd(d, xt, wt))
    xb, wb, _, d = make(rng, dev, M, N, K, torch.bfloat16, layout, False, True)      # d_x [M,N]
    check_bwd(xb, wb, d, None, "none", ops.dense_bwd(d, xb, wb))


@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_float32_output_and_float32_upstream_gradient(dev, name):
    from objectdetection_amd import ops
    x, w, b, _ = make(np.random.default_rng(3), dev, 70, 520, 21, TYPES[name], "nk")
    out = ops.dense_fwd(x, w, b, out_dtype=torch.float32)
    assert out.dtype == torch.float32
    check_fwd(x, w, b, None, "none", out, odt=torch.float32)
    d = torch.randn((70, 21), device=dev)
    check_bwd(x, w, d, None, "none", ops.dense_bwd(d, x, w))


def test_rows_with_strides_slices_and_pooled_shape(dev):
    """Column slices (strided rows, odd alignments), sliced weights, an expanded gradient, 5-D and 3-D x."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(5)
    big, _, b, _ = make(rng, dev, 90, 260, 45, torch.bfloat16)
    wide = make(rng, dev, 200, 200, 64, torch.bfloat16)[1]
    for c0, k in ((0, 128), (1, 131), (8, 200)):
        x, w = big[:, c0:c0 + k], wide[:k, 3:48]
        check_fwd(x, w, b, None, "relu", ops.dense_fwd(x, w, b, act="relu"))
        d = big[:, 7:52]
        check_bwd(x, w, d, None, "none", ops.dense_bwd(d, x, w))
        one = torch.ones((1, 1), dtype=torch.bfloat16, device=dev).expand(90, 45)       # .sum()'s gradient
        check_bwd(x, w, one, None, "none", ops.dense_bwd(one, x, w))
    x, w, b, res = make(rng, dev, 12, 7 * 7 * 8, 40, torch.float16, "nk", True, True)
    out = ops.dense_fwd(x.view(3, 4, 7, 7, 8), w, b, "silu", res.view(3, 4, 40))
    assert out.shape == (3, 4, 40)
    check_fwd(x, w, b, res, "silu", out)
    assert torch.equal(out.view(12, 40), ops.dense_fwd(x, w, b, "silu", res))
    g = ops.dense_bwd(res.view(3, 4, 40), x.view(3, 4, 7, 7, 8), w)
    assert g["d_x"].shape == (3, 4, 7, 7, 8)
    check_bwd(x, w, res, None, "none", g)
    assert ops.dense_fwd(x.view(2, 2, 3, 392), w).shape == (2, 2, 3, 40)
    x1, x3 = x[:, 0].contiguous(), x[:, 3:4]                     # one feature; a [K] vector as one row
    assert torch.equal(ops.dense_fwd(x3, w[3:4]), ops.dense_fwd(x3.contiguous(), w[3:4].contiguous()))
    check_fwd(x1.view(1, 12), w[:12], None, None, "none", ops.dense_fwd(x1, w[:12]))


def test_no_rows(dev):
    from objectdetection_amd import ops
    x, w, b, _ = make(np.random.default_rng(5), dev, 4, 24, 9, torch.bfloat16)
    out, pre = ops.dense_fwd(x[:0], w, b, act="gelu", want_pre=True)
    assert out.shape == (0, 9) and pre.shape == (0, 9)
    for ww in (w, w.t().contiguous().t()):
        g = ops.dense_bwd(out, x[:0], ww, pre=pre, act="gelu")
        assert g["d_x"].shape == (0, 24) and not g["d_weight"].any() and not g["d_bias"].any()
        assert g["d_weight"].shape == (24, 9)


def test_rows_and_columns_outside_the_result_stay(dev):
    """`out` as the rows of a larger buffer: what lies behind the last row and value is not written."""
    from objectdetection_amd import ops
    for M, K, N in ((5, 40, 13), (131, 520, 130), (1, 4096, 24)):
        x, w, b, _ = make(np.random.default_rng(M), dev, M, K, N, torch.bfloat16)
        buf = torch.full((M * N + 300,), 7.0, dtype=torch.bfloat16, device=dev)
        ops.dense_fwd(x, w, b, out=buf[:M * N].view(M, N))
        check_fwd(x, w, b, None, "none", buf[:M * N].view(M, N))
        assert (buf[M * N:] == 7).all()


def test_infinities_and_nan(dev):
    from objectdetection_amd import ops
    inf, nan = math.inf, math.nan
    eye = torch.eye(8, device=dev, dtype=torch.bfloat16)
    row = torch.tensor([[0.0, 1, -1, 3e38, -3e38, 5, -5, 0.5]], device=dev).bfloat16()
    for act in ("relu", "gelu", "silu"):
        got = ops.dense_fwd(row, eye, act=act)
        ref = act64(f64(row), act)
        assert torch.allclose(got.double().cpu(), ref, rtol=2 ** -7, atol=1e-7), act
    bias = torch.tensor([inf, -inf, nan, 0, 1, -1, 2, -2], device=dev).bfloat16()
    z = torch.zeros((1, 8), device=dev, dtype=torch.bfloat16)
    got = ops.dense_fwd(z, eye, bias, act="relu").float().cpu()
    assert got[0, 0] == inf and got[0, 1] == 0 and got[0, 2].isnan() and not got[0, 3:].isnan().any()
    g = ops.dense_bwd(torch.full((1, 8), inf, device=dev).bfloat16(), z, eye, pre=bias[None], act="relu")
    assert g["d_bias"].float().cpu().tolist() == [inf, 0, 0, 0, inf, 0, inf, 0]
    # a NaN row or column reaches its own results only, also where tiles are padded
    x, w, b, _ = make(np.random.default_rng(1), dev, 19, 70, 37, torch.float16)
    x[7] = nan
    w = w.clone()
    w[:, 5] = inf
    out = ops.dense_fwd(x, w, b)
    bad = ~out.isfinite()
    ref = torch.zeros_like(bad)
    ref[7] = True
    ref[:, 5] = True
    assert torch.equal(bad, ref)


@pytest.mark.parametrize("M", [3, 70])
def test_values_below_the_normal_range(dev, M):
    """float16 subnormals are kept as operands and as results (a factor of two exact)."""
    from objectdetection_amd import ops
    x = (2.0 ** -24 * torch.arange(1, M + 1, device=dev)).half()[:, None] * torch.eye(8, device=dev)[0].half()
    w = torch.full((8, 16), 2.0, device=dev).half()
    for ww in (w, w.t().contiguous().t()):
        assert torch.equal(ops.dense_fwd(x, ww), (2.0 ** -23 * torch.arange(1, M + 1, device=dev)).half()[:, None].expand(M, 16))
        d = torch.zeros((M, 16), device=dev).half()
        d[:, 3] = 2.0 ** -24
        assert (ops.dense_bwd(d, x, ww)["d_x"] == 2.0 ** -23).all()


def test_a_workspace_is_written_before_it_is_read(dev):
    """A workspace full of NaN, and one byte more than needed behind it, change nothing."""
    from objectdetection_amd import ops
    for M, K, N, layout in ((1, 25088, 24, "kn"), (130, 1003, 333, "nk"), (90, 8200, 84, "kn"), (5000, 40, 84, "nk")):
        x, w, b, d = make(np.random.default_rng(7), dev, M, K, N, torch.bfloat16, layout, True, True)
        lay = 0 if layout == "kn" else 1
        pre = ops.dense_fwd(x, w, b, want_pre=True)[1]
        nf, nb = ops.dense_fwd_workspace_bytes(M, K, N, lay), ops.dense_bwd_workspace_bytes(M, K, N, lay)
        ws = torch.full((max(nf, nb) + 256,), 255, dtype=torch.uint8, device=dev)
        assert torch.equal(ops.dense_fwd(x, w, b, workspace=ws[:nf] if nf else None), ops.dense_fwd(x, w, b))
        assert (ws[nf:] == 255).all()
        ws.fill_(255)
        g, h = ops.dense_bwd(d, x, w, pre, "silu", workspace=ws[:nb]), ops.dense_bwd(d, x, w, pre, "silu")
        assert all(torch.equal(g[k], h[k]) for k in g) and (ws[nb:] == 255).all()


def test_only_the_wanted_gradients(dev):
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(8), dev, 300, 203, 85, torch.float16, "nk", True, True)
    pre = ops.dense_fwd(x, w, b, want_pre=True)[1]
    full = ops.dense_bwd(d, x, w, pre, "gelu")
    for n in range(1, 8):
        g = ops.dense_bwd(d, x, w, pre, "gelu", bool(n & 1), bool(n & 2), bool(n & 4))
        for bit, key in ((1, "d_x"), (2, "d_weight"), (4, "d_bias")):
            assert torch.equal(g[key], full[key]) if n & bit else g[key] is None


def test_same_bits_every_time_and_on_another_stream(dev):
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(9), dev, 40, 4104, 84, torch.bfloat16, "nk", True, True)
    out, g = ops.dense_fwd(x, w, b), ops.dense_bwd(d, x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(out, ops.dense_fwd(x, w, b))
            h = ops.dense_bwd(d, x, w)
            assert all(torch.equal(g[k], h[k]) for k in g)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("M,K,N,layout", [(24, 2056, 136, "kn"), (130, 1003, 333, "nk"), (4100, 72, 2056, "kn"),
                                          (700, 4096, 84, "nk")])
def test_captured_forward_and_backward_replay(dev, M, K, N, layout):
    """Two graphs of the same calls with a workspace each, replayed with other work between: few rows,
    packed operands, the large tile, a split reduction."""
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(11), dev, M, K, N, torch.bfloat16, layout, True, True)
    lay = 0 if layout == "kn" else 1
    ws = [torch.empty(max(16, ops.dense_fwd_workspace_bytes(M, K, N, lay), ops.dense_bwd_workspace_bytes(M, K, N, lay)),
                      dtype=torch.uint8, device=dev) for _ in range(2)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for n in range(2):
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, pre = ops.dense_fwd(x, w, b, act="gelu", want_pre=True, workspace=ws[n])
            g = ops.dense_bwd(d, x, w, pre=pre, act="gelu", workspace=ws[n])
        graphs.append(graph)
        outs.append((out, g))
    for step in range(4):
        x.copy_(torch.randn_like(x))
        for n in range(2):
            graphs[n].replay()
        torch.cuda.synchronize()
        ref, pre = ops.dense_fwd(x, w, b, act="gelu", want_pre=True)
        gref = ops.dense_bwd(d, x, w, pre=pre, act="gelu")
        for out, g in outs:
            assert torch.equal(out, ref) and all(torch.equal(g[k], gref[k]) for k in g), step


def test_gradients_against_differences(dev):
    """d_x, d_weight, d_bias of sum(d_out * out) against central differences in float64 of the formula,
    through act' at the saved pre-activations."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(2)
    for act in ("gelu", "silu"):
        x, w, b, d = make(rng, dev, 6, 16, 8, torch.float16, "kn", True, True)
        out, pre = ops.dense_fwd(x, w, b, act=act, want_pre=True)
        g = ops.dense_bwd(d, x, w, pre=pre, act=act)
        X, W, B, D = f64(x), f64(w), f64(b), f64(d)
        f = lambda X, W, B: float((D * act64(X @ W + B, act)).sum())
        h = 1e-4
        for t, got, call in ((X, g["d_x"], lambda t: f(t, W, B)), (W, g["d_weight"], lambda t: f(X, t, B)),
                             (B, g["d_bias"], lambda t: f(X, W, t))):
            num = torch.zeros_like(t)
            for i in range(t.numel()):
                p, m = t.clone().view(-1), t.clone().view(-1)
                p[i] += h
                m[i] -= h
                num.view(-1)[i] = (call(p.view(t.shape)) - call(m.view(t.shape))) / (2 * h)
            # float16: pre, dz and the result are rounded (2^-11 each, relative to the absolute sums)
            assert (f64(got) - num).abs().max() <= 4 * 2.0 ** -11 * max(1.0, float(num.abs().max())) * 4


def test_refusals(dev):
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(1), dev, 4, 24, 8, torch.bfloat16, "kn", True, True)
    for bad, err in (
            (lambda: ops.dense_fwd(x.float(), w.float()), TypeError),
            (lambda: ops.dense_fwd(x, w.half()), TypeError),
            (lambda: ops.dense_fwd(x, w[:20]), ValueError),
            (lambda: ops.dense_fwd(x, w[0]), ValueError),
            (lambda: ops.dense_fwd(x, w, b.float()), TypeError),
            (lambda: ops.dense_fwd(x, w, b[:7]), ValueError),
            (lambda: ops.dense_fwd(x, w, act="tanh"), ValueError),
            (lambda: ops.dense_fwd(x, w, residual=d[:1]), ValueError),
            (lambda: ops.dense_fwd(x, w, residual=d.float()), TypeError),
            (lambda: ops.dense_fwd(x, w, out=torch.empty((4, 8), device=dev)), ValueError),
            (lambda: ops.dense_fwd(x, w, out_dtype=torch.float16), TypeError),
            (lambda: ops.dense_fwd(x.cpu(), w), RuntimeError),
            (lambda: ops.dense_fwd(x, w.cpu()), RuntimeError),
            (lambda: ops.dense_bwd(d, x, w, act="relu"), ValueError),
            (lambda: ops.dense_bwd(d[:3], x, w), ValueError),
            (lambda: ops.dense_bwd(d, x, w, want_dx=False, want_dw=False, want_db=False), ValueError),
            (lambda: ops.dense_bwd(d, x, w, pre=d, act="relu", workspace=torch.empty(16, dtype=torch.uint8, device=dev)),
             ValueError)):
        with pytest.raises(err):
            bad()


def test_the_output_may_be_the_residual_and_nothing_else(dev):
    from objectdetection_amd import ops
    rng = np.random.default_rng(15)
    for M, K, N in ((5, 40, 13), (5, 40, 45), (20, 9000, 47), (300, 136, 136), (3000, 64, 520), (60, 8200, 84)):
        x, w, b, d = make(rng, dev, M, K, N, torch.bfloat16, "nk", True, True)
        ref = ops.dense_fwd(x, w, b, "silu", residual=d)
        assert ops.dense_fwd(x, w, b, "silu", residual=d, out=d) is d and torch.equal(d, ref)
    x, w, b, d = make(rng, dev, 40, 40, 40, torch.bfloat16, "kn", True, True)
    for bad in (x, w, w.t(), b):
        out = torch.as_strided(bad, (40, 40), (40, 1), bad.storage_offset()) if bad is not b else None
        if out is None:
            store = torch.zeros(1600, dtype=torch.bfloat16, device=dev)
            b, out = store[80:120], store.view(40, 40)
        with pytest.raises(ValueError, match="overlaps"):
            ops.dense_fwd(x, w, b, out=out)
    two = torch.zeros((41, 40), dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="overlaps residual"):
        ops.dense_fwd(x, w, b, residual=two[:40], out=two[1:])


def test_rows_further_apart_than_32_bits(dev):
    """Row strides of 2,097,152 elements: the last rows lie 4.3 GB behind the first."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(16)
    M, K, N, ld = 1030, 72, 40, 1 << 21
    x, w, b, d = make(rng, dev, M, K, N, torch.bfloat16, "nk", True, True)
    buf = torch.empty((M * ld,), dtype=torch.bfloat16, device=dev)
    far = lambda at, n: torch.as_strided(buf, (M, n), (ld, 1), at)
    far(0, K).copy_(x)
    far(128, N).copy_(d)
    for act in ("none", "gelu"):
        out, pre = ops.dense_fwd(far(0, K), w, b, act, residual=far(128, N), want_pre=True)
        ref = ops.dense_fwd(x, w, b, act, residual=d, want_pre=True)
        assert torch.equal(out, ref[0]) and torch.equal(pre, ref[1])
        g, h = ops.dense_bwd(far(128, N), far(0, K), w, pre, act), ops.dense_bwd(d, x, w, pre, act)
        assert all(torch.equal(g[k], h[k]) for k in g)
    # the few rows' kernel, a weight of rows as far apart
    wide = torch.as_strided(buf, (K, M), (1, ld), 0)          # Linear weight [1030, 72]
    assert torch.equal(ops.dense_fwd(x[:20], wide), ops.dense_fwd(x[:20], x.t()))


def test_two_streams_at_once(dev):
    """Calls of different sizes queued on two streams give what they give one after the other."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(17)
    cases = [make(rng, dev, *s, torch.bfloat16, "nk", True, True) for s in
             ((700, 4096, 84), (130, 1003, 333), (4100, 72, 2056), (24, 2056, 136))]
    z = torch.randn((70, 40000), device=dev)
    t, i = torch.randn((70, 8), device=dev), torch.randint(0, 40000, (70, 8), device=dev)

    def work(case):
        x, w, b, d = case
        out, pre = ops.dense_fwd(x, w, b, "gelu", want_pre=True)
        g = ops.dense_bwd(d, x, w, pre, "gelu")
        o = ops.distill_loss(z, t, i, temperature=2.0)
        return [out, pre, *g.values(), *o.values()]

    want = [work(c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for n, c in enumerate(cases):
            with torch.cuda.stream(streams[n % 2]):
                got.append((n, work(c)))
    torch.cuda.synchronize()
    for n, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[n])), n


@pytest.mark.parametrize("M,K,N", [(3, 4104, 2056), (17, 4104, 2056), (32, 8200, 4104)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_few_rows_of_large_weights(dev, M, K, N, layout):
    """Up to 32 rows: weights in whole pieces go through the tiles when they are large, others as they are."""
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(M), dev, M, K, N, torch.bfloat16, layout, True, True)
    odd = torch.zeros((K * N + 1,), dtype=torch.bfloat16, device=dev)[1:]
    odd = odd.view(w.t().shape).t() if layout == "nk" else odd.view(w.shape)
    odd.copy_(w)
    lay = 0 if layout == "kn" else 1
    for ww in (w, odd):
        out, pre = ops.dense_fwd(x, ww, b, "gelu", residual=d, want_pre=True)
        check_fwd(x, w, b, d, "gelu", out, pre)
        most = torch.empty(max(16, ops.dense_fwd_workspace_bytes(M, K, N, lay)), dtype=torch.uint8, device=dev)
        assert torch.equal(ops.dense_fwd(x, ww, b, "gelu", residual=d, workspace=most), out)
        check_bwd(x, w, d, pre, "silu", ops.dense_bwd(d, x, ww, pre, "silu"))
    shifted = torch.empty((M * K + 3,), dtype=torch.bfloat16, device=dev)[3:].view(M, K)
    shifted.copy_(x)                                       # rows that do not start on 16 bytes
    ref = ops.dense_fwd(x, w, b)
    most = torch.full((max(16, ops.dense_fwd_workspace_bytes(M, K, N, lay)) + 64,), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(ops.dense_fwd(shifted, w, b, workspace=most[:-64]), ref) and (most[-64:] == 255).all()
    g, h = ops.dense_bwd(d, shifted, w), ops.dense_bwd(d, x, w)
    assert all(torch.equal(g[k], h[k]) for k in g)


@pytest.mark.parametrize("M,K,N", [(1111, 779, 333), (300, 203, 85), (64, 512, 512), (257, 16, 8), (40, 40, 40), (1000, 136, 1000)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_small_backward_in_one_launch_gives_the_same_bits(dev, M, K, N, layout):
    """Both products and the bias gradient of a small backward share launches; asked for one by one they do not."""
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(M), dev, M, K, N, torch.float16, layout, True, True)
    pre = ops.dense_fwd(x, w, b, want_pre=True)[1]
    for act in ("silu", "none"):
        full = ops.dense_bwd(d, x, w, pre, act)
        check_bwd(x, w, d, pre, act, full)
        for key, want in (("d_x", (True, False, False)), ("d_weight", (False, True, False)), ("d_bias", (False, False, True))):
            assert torch.equal(ops.dense_bwd(d, x, w, pre, act, *want)[key], full[key]), key
        two = ops.dense_bwd(d, x, w, pre, act, want_db=False)
        assert torch.equal(two["d_x"], full["d_x"]) and torch.equal(two["d_weight"], full["d_weight"])
        lay = 0 if layout == "kn" else 1
        ws = torch.full((ops.dense_bwd_workspace_bytes(M, K, N, lay) + 256,), 255, dtype=torch.uint8, device=dev)
        g = ops.dense_bwd(d, x, w, pre, act, workspace=ws[:-256])
        assert all(torch.equal(g[k], full[k]) for k in g) and (ws[-256:] == 255).all()


@pytest.mark.parametrize("M,K,N", [(1, 4096, 21), (9, 4103, 5), (32, 2048, 31), (3, 70, 1), (20, 9000, 3), (2, 64, 30), (4, 71, 9)])
def test_few_rows_of_a_narrow_kernel(dev, M, K, N):
    """Fewer than 32 columns: what is loaded beside them never reaches a result (infinities and NaN around the matrix)."""
    from objectdetection_amd import ops
    x, w, b, d = make(np.random.default_rng(K), dev, M, K, N, torch.float16, "kn", True, True)
    for ld in (N, N + 3, N + 40):
        wide = torch.full((K * ld + 64,), math.nan, dtype=torch.float16, device=dev)
        ww = torch.as_strided(wide, (K, N), (ld, 1), 32)
        ww.copy_(w)
        check_fwd(x, w, b, d, "relu", ops.dense_fwd(x, ww, b, "relu", residual=d))
        end = torch.empty((K * ld,), dtype=torch.float16, device=dev)
        last = torch.as_strided(end, (K, N), (ld, 1), ld - N)          # its last value is the buffer's
        last.copy_(w)
        assert torch.equal(ops.dense_fwd(x, last, b), ops.dense_fwd(x, w, b))


def test_first_calls_inside_a_capture(dev):
    """Sizes whose kernels no other test has launched yet in this type and layout: the first call is captured."""
    from objectdetection_amd import ops
    rng = np.random.default_rng(31)
    for M, K, N, layout in ((333, 264, 200, "kn"), (2100, 520, 2100, "nk")):
        x, w, b, d = make(rng, dev, M, K, N, torch.bfloat16, layout, True, True)
        pre = torch.randn((M, N), device=dev).bfloat16()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = ops.dense_fwd(x, w, b, "silu", residual=d)
            grads = ops.dense_bwd(d, x, w, pre, "silu")
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            check_fwd(x, w, b, d, "silu", out)
            check_bwd(x, w, d, pre, "silu", grads)
            ref = ops.dense_bwd(d, x, w, pre, "silu")
            assert all(torch.equal(ref[k], grads[k]) for k in ref) and torch.equal(out, ops.dense_fwd(x, w, b, "silu", residual=d))
            for t in (out, *grads.values()):
                t.zero_()
