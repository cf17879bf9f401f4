"""GELU over its whole range, the negative tail relative to itself (float32 output).

Phi is a polynomial (1.3e-6 relative in float32) times e^(-z^2/2) in two parts, exp2 and rcp within 1 ulp (2^-23) each,
and three products (2^-24 each): below 2e-6 of z Phi(z), as far down as that is a normal number."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 70])
def test_the_tail_relative_to_itself(dev, name, rows):
    from objectdetection_amd import ops
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[name]
    z = torch.cat([torch.linspace(-12.8, 0, 4000), torch.linspace(0, 12, 1000), -2.0 ** torch.arange(-14.0, 3.0)]).to(dt)
    z = torch.cat([z, z.new_zeros(-z.numel() % rows)]).view(rows, -1).to(dev)
    n = z.shape[1]
    eye = torch.eye(n, device=dev).to(dt)
    for w in (eye, eye.t().contiguous().t()):
        got = ops.dense_fwd(z, w, act="gelu", out_dtype=torch.float32).double().cpu()
        ref = torch.tensor([v * 0.5 * math.erfc(-v / math.sqrt(2)) for v in z.double().cpu().flatten().tolist()]).view(got.shape).double()
        off = (got - ref).abs()
        assert (off <= 2e-6 * ref.abs() + 2.0 ** -126).all(), float((off / ref.abs()).nan_to_num(nan=0.0).max())


def test_far_values(dev):
    """Where e^(-z^2/2) is 0 and z^2 beyond float32; NaN stays."""
    from objectdetection_amd import ops
    z = torch.tensor([[-3e38, -1e20, -20, -14.5, 14.5, 1e20, 3e38, math.inf, math.nan]], device=dev).bfloat16()
    for M in (1, 40):
        x, w = torch.zeros((M, 9), device=dev).bfloat16(), torch.zeros((9, 9), device=dev).bfloat16()
        got = ops.dense_fwd(x, w, z[0], "gelu", out_dtype=torch.float32)
        assert not got[:, :4].any() and torch.equal(got[:, 4:8], z[:, 4:8].float().expand(M, 4)) and got[:, 8].isnan().all()
        g = ops.dense_bwd(torch.ones_like(x), x, torch.eye(9, device=dev).bfloat16(), z.repeat(M, 1), "gelu")["d_bias"]
        assert not g[:4].any() and (g[4:7] == M).all() and g[8].isnan()
