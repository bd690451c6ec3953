"""The norm and rows in 8 bits where a value, a place in memory or a width is out of the ordinary.  Bounds as in
test_gpu_residual_norm.py."""
import pytest
import torch

from graphiler_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
STEPS = 42 * 2.0 ** -24
EPS = 1e-6


def make(seed, rows, cols, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen))
    r, gy = torch.randn(rows, cols, generator=gen), 0.1 * torch.randn(rows, cols, generator=gen)
    w = 1 + 0.3 * torch.randn(cols, generator=gen)
    return tuple(t.to(dtype).cuda() for t in (x, r, w, gy))


def within(got, want, bound):
    worst = ((got.double() - want).abs() / (bound + 1e-300)).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(5, 300), (3, 1000), (3, 3000), (2, 16384)])
@pytest.mark.parametrize("power,eps", [(53, EPS), (-53, 0.0)])
def test_gradients_of_rows_of_any_size(rows, cols, dtype, power, eps):
    """Rows about 1e16 or 1e-16: 1 / sqrt(mean) is in range, its cube is not."""
    x, _, w, gy = make(rows + cols, rows, cols, dtype)
    x = x * 2.0 ** power
    gx, gw = ops.rms_norm_backward(gy, x, w, eps)
    t, g, v = x.double(), gy.double(), w.double()
    inv = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + eps)
    dot = (t * inv * v * g).mean(1, keepdim=True)
    want = inv * (v * g - t * inv * dot)
    size = inv * ((v * g).abs() + (t * inv).abs() * (t * inv * v * g).abs().mean(1, keepdim=True))
    half_step = torch.finfo(dtype).eps / 2
    # a term is three or four roundings and powers of the root: each is off by at most 4 STEPS
    within(gx, want, 4 * STEPS * size + (half_step + 2.0 ** -24) * want.abs())
    terms = (g * t * inv).abs().sum(0)
    within(gw, (g * t * inv).sum(0), (rows * 2.0 ** -24 + 2 * STEPS) * terms + half_step * terms)
