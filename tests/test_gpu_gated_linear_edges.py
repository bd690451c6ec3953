"""The gated block and its gradients where test_gpu_gated_linear.py does not go: infinities, operands at any address,
every activation in every tile.  Bounds and the plain forms are that file's."""
import math

import pytest
import torch
from test_gpu_gated_linear import ACTS, DTYPES, check_backward, make

from graphiler_amd import ops

pytestmark = pytest.mark.gpu

# rows, K, F; whether fp32 products of this size are formed by the fp32 instruction, as few rows, few columns and up to 1024
# tiles of 64 x 32 are for K <= 256 (43 x 22 tiles of 2720 x 704, 47 x 32 of 3000 x 1000), else of pieces.  bf16: few rows,
# tiles of 64, 64, 128 and 256 rows.
SIZES = [(6, 100, 90, True), (16, 72, 130, True), (200, 100, 90, True), (2720, 256, 704, True), (3000, 72, 1000, False),
         (3840, 72, 1664, False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,k,f,instruction", SIZES)
def test_an_infinity_of_a_row(rows, k, f, instruction, act, dtype):
    """x[4, k - 1] = inf: gate and up are infinities of their weights' signs.  act(inf) up has up's sign; act(-inf) is 0
    times an infinity, or NaN already.  Products of pieces give NaN."""
    x, wg, wu, _ = make(rows, rows, k, f, dtype)
    clean = ops.gated_linear(x, wg, wu, act)
    x[4, k - 1] = math.inf
    assert not bool((wg[k - 1] == 0).any()) and not bool((wu[k - 1] == 0).any())
    h = ops.gated_linear(x, wg, wu, act)
    keep = [i for i in range(rows) if i != 4]
    assert torch.equal(h[keep], clean[keep])
    up = wg[k - 1] > 0
    if dtype == torch.bfloat16 or instruction:
        assert torch.equal(h[4, up].float(), torch.sign(wu[k - 1, up].float()) * math.inf)
        assert bool(torch.isnan(h[4, ~up]).all())
    else:
        assert bool(torch.isnan(h[4]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("rows,k,f", [(300, 40, 700), (3600, 72, 1800), (700, 1800, 1900), (8192, 1280, 40), (70, 2048, 2600)])
def test_gradients_of_activations_in_all_tiles(rows, k, f, dtype, act):
    check_backward(rows, k, f, dtype, act)


def moved(t):
    """The same values one element further on than an allocation begins."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(40, 64, 64), (300, 96, 700), (3600, 72, 1800)])
def test_a_gradient_at_any_address(rows, k, f, dtype):
    """grad_h whose rows are whole groups of four, but not at 8 or 16 bytes: read value by value."""
    x, wg, wu, gh = make(rows + f, rows, k, f, dtype)
    want = ops.gated_linear_backward(gh, x, wg, wu, "gelu")
    got = ops.gated_linear_backward(moved(gh), x, wg, wu, "gelu")
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(3, 65, 67), (16, 1003, 130), (40, 75, 133), (3001, 75, 133)])
def test_operands_at_any_address(rows, k, f, dtype):
    """Rows that are not whole 16-byte pieces may begin anywhere."""
    x, wg, wu, gh = make(rows + f, rows, k, f, dtype)
    assert torch.equal(ops.gated_linear(moved(x), moved(wg), moved(wu)), ops.gated_linear(x, wg, wu))
    for a, b in zip(ops.gated_linear_backward(moved(gh), moved(x), moved(wg), moved(wu)),
                    ops.gated_linear_backward(gh, x, wg, wu)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(1, 64, 64), (9, 256, 512), (16, 1024, 136)])
def test_few_rows_at_any_address(rows, k, f, dtype):
    """Rows that are whole 16-byte pieces too, as long as there are few."""
    x, wg, wu, _ = make(rows + f, rows, k, f, dtype)
    want = ops.gated_linear(x, wg, wu)
    for i in range(3):
        args = [x, wg, wu]
        args[i] = moved(args[i])
        assert torch.equal(ops.gated_linear(*args), want)
    gh = torch.randn_like(want)
    leaves = [moved(t).requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(ops.gated_linear(*leaves), leaves, moved(gh))
    for a, b in zip(got, ops.gated_linear_backward(gh, x, wg, wu)):
        assert torch.equal(a, b)
    x = make(1, 17, k, f, dtype)[0]
    if dtype == torch.bfloat16:
        with pytest.raises(RuntimeError, match="(?i)align"):
            ops.gated_linear(moved(x), wg, wu)
    else:
        assert torch.equal(ops.gated_linear(moved(x), wg, wu), ops.gated_linear(x, wg, wu))
