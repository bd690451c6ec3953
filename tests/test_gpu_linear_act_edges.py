"""Projections where test_gpu_linear_act.py does not go: values that are not finite."""
import math

import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import ops
from test_gpu_linear_act import DEV, HALF_STEP, U, made, operands, product_bound, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("rows,k,m", [(5, 40, 9), (33, 64, 64), (33, 64, 65), (200, 72, 70), (130, 100, 4), (600, 64, 1023)])
def test_an_infinity_of_a_row_leaves_its_gradient_finite(rows, k, m, bad, act):
    """x[3, 1] = +-inf: z of that row is infinite, its slope 0 or 1, so dz and grad_x are finite, for any number of columns.
    bf16: an fp32 operand that is not finite gives NaN."""
    dtype, r = torch.bfloat16, HALF_STEP[torch.bfloat16]
    x, w, b, _ = operands(rows, k, m, dtype, True, False)
    w[1][w[1] == 0] = 1.0
    x[3, 1] = bad
    gy = made((rows, m), dtype, 5, 0.1)
    gx, gw, gb = ops.linear_act_backward(gy, x, w, bias=b, activation=act)
    tame = x.double()
    tame[3, 1] = 0
    wd, gd = w.double(), gy.double()
    z = tame @ wd + b.double()
    z_off = product_bound(tame, wd) + 2 * U * z.abs()
    z[3], z_off[3] = wd[1].sign() * bad, 0
    if act == "relu":
        slope = (z > 0).double()
        off = torch.where(z.abs() <= z_off, gd.abs(), 2 * U * gd.abs())
    else:
        density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        slope = 0.5 * torch.erfc(-z / math.sqrt(2)) + torch.where(density > 0, z, torch.zeros_like(z)) * density
        size = torch.where(z.isfinite(), z.abs(), torch.zeros_like(z))
        off = gd.abs() * (z_off + 2.0 ** -20 * (size + 8))
    dz = gd * slope
    off = off + r * (dz.abs() + off)
    want, tol = dz @ wd.t(), off @ wd.t().abs() + product_bound(dz, wd.t())
    within(gx, want, tol + r * (want.abs() + tol) + 1e-37, "gradient of x")
    want, tol = dz.sum(0), off.sum(0) + (rows + 8) * U * dz.abs().sum(0)
    within(gb, want, tol + r * (want.abs() + tol) + 1e-37, "gradient of the bias")
    want, tol = tame.t() @ dz, tame.t().abs() @ off + product_bound(tame.t(), dz)
    others = [i for i in range(k) if i != 1]                 # row 1 sums multiples of the infinity
    within(gw[others], want[others], (tol + r * (want.abs() + tol) + 1e-37)[others], "gradient of weight")


def test_the_slope_of_silu_at_an_infinity_is_its_columns_own():
    """silu's slope is s + z s (1 - s), inf x 0 at +inf and at -inf: NaN wherever it is formed, and nowhere else."""
    for m in (64, 65):
        x, w, b, _ = operands(40, 64, m, torch.bfloat16, True, False)
        x[3, 1] = math.inf
        gx, _, _ = ops.linear_act_backward(made((40, m), torch.bfloat16, 5), x, w, bias=b, activation="silu")
        assert torch.isnan(gx[3]).all() and torch.isfinite(gx[torch.arange(40, device=DEV) != 3]).all()
