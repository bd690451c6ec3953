"""The norm and rows in 8 bits where a value, a place in memory or a width is out of the ordinary.  Bounds as in
test_gpu_residual_norm.py."""
import pytest
import torch

from graphiler_amd import capi, layers, ops

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(33, 100), (9, 500), (7, 1000), (5, 2000), (5, 4096), (4, 7000), (3, 16384)])
def test_results_in_place_of_operands(rows, cols, dtype):
    """sum over x or over the residual, grad_x over grad_y or over grad_sum: the same bits as beside them."""
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    dt = capi.GA_F32 if dtype == torch.float32 else capi.GA_BF16
    x, r, w, gy = make(cols, rows, cols, dtype)
    y, t = ops.rms_norm(x, w, r, EPS)
    y8, scales, _ = ops.rms_norm_fp8(x, w, r, EPS)
    for over in ("x", "residual"):
        a, b = x.clone(), r.clone()
        total, mine = a if over == "x" else b, torch.empty_like(y)
        assert lib.ga_rms_norm(a.data_ptr(), b.data_ptr(), w.data_ptr(), mine.data_ptr(), total.data_ptr(), rows, cols,
                               EPS, dt, stream) == 0
        assert torch.equal(mine, y) and torch.equal(total, t)
        a, b = x.clone(), r.clone()
        total, mine8, mine_scales = a if over == "x" else b, torch.empty_like(y8), torch.empty_like(scales)
        assert lib.ga_rms_norm_fp8(a.data_ptr(), b.data_ptr(), w.data_ptr(), mine8.data_ptr(), mine_scales.data_ptr(),
                                   total.data_ptr(), rows, cols, EPS, dt, stream) == 0
        assert torch.equal(total, t) and torch.equal(mine8.view(torch.uint8), y8.view(torch.uint8))
        assert torch.equal(mine_scales.view(torch.uint8), scales.view(torch.uint8))
    n = lib.ga_rms_norm_backward_workspace_bytes(rows, cols)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    for gt in (None, r):
        gx, gw = ops.rms_norm_backward(gy, t, w, EPS, gt)
        for over in ("grad_y", "grad_sum"):
            if gt is None and over == "grad_sum":
                continue
            a, b, mine = gy.clone(), None if gt is None else gt.clone(), torch.empty_like(gw)
            out = a if over == "grad_y" else b
            assert lib.ga_rms_norm_backward(a.data_ptr(), t.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(),
                                            out.data_ptr(), mine.data_ptr(), rows, cols, EPS, dt, ws.data_ptr(), n,
                                            stream) == 0
            assert torch.equal(out, gx) and torch.equal(mine, gw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 100, 129, 300, 1000, 2047, 5001])
def test_zeros_behind_rows_that_are_not_finite(cols, dtype):
    x, r, w, _ = make(cols, 4, cols, dtype)
    x[1, 0], x[2, cols - 1], x[3], r[3] = float("nan"), float("inf"), 0.0, 0.0
    for residual in (None, r):
        y8, scales = ops.rms_norm_fp8(x, w, residual, eps=0.0)[:2]
        assert bool((y8[:, cols:].view(torch.uint8) == 0).all())
        y = ops.rms_norm(x, w, residual, eps=0.0)
        y = y if residual is None else y[0]
        assert torch.equal(torch.isnan(y8[:, :cols].float()), ~torch.isfinite(y))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [16385, 20001, 32640, 32768])
def test_rows_as_wide_as_the_8_bit_products_are_cut(cols, dtype):
    """Blocks of 128 are cut by themselves: the same bits as two narrower halves."""
    x = make(cols, 3, cols, dtype)[0]
    x[1, cols - 1] = float("inf")
    x8, scales = ops.quantize_fp8(x)
    assert x8.shape == (3, -(-cols // 128) * 128) and scales.shape == (3, -(-cols // 128))
    for part in (slice(0, 16384), slice(16384, cols)):
        a8, a_scales = ops.quantize_fp8(x[:, part].contiguous())
        blocks = slice(part.start // 128, part.start // 128 + a_scales.shape[1])
        assert torch.equal(x8[:, part.start:part.start + a8.shape[1]].view(torch.uint8), a8.view(torch.uint8))
        assert torch.equal(scales[:, blocks].view(torch.uint8), a_scales.view(torch.uint8))


def test_a_block_as_wide_as_the_8_bit_products():
    gen = torch.Generator().manual_seed(5)
    for f in (16385, 32768):
        x = torch.randn(5, 64, generator=gen).cuda()
        w = [torch.randn(64, f, generator=gen).cuda() / 8 for _ in range(2)] + [torch.randn(f, 32, generator=gen).cuda() / f ** 0.5]
        w8 = [ops.quantize_weight_fp8(t) for t in w]
        got = layers.feed_forward(x, *w8)
        hidden = ops.gated_linear_fp8(*ops.quantize_fp8(x), *w8[0], *w8[1], out_dtype=torch.float32)

        def held(values, scales, rows_each):             # what the 8 bits stand for
            s = torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(rows_each, 0)[:values.shape[0]]
            return values.double() * s.repeat_interleave(128, 1)

        h, down = held(*ops.quantize_fp8(hidden), 1), held(*w8[2], 128)
        want, size = h @ down.t(), h.abs() @ down.t().abs()
        # of eight products what is 2^-13 below the largest is dropped, then f sums in fp32, one rounding
        assert ((got.double() - want).abs() <= (2.0 ** -10 + f * 2.0 ** -24) * size + 2.0 ** -24 * want.abs()).all()
        with pytest.raises(RuntimeError, match="at most 32768 columns"):
            ops.quantize_fp8(torch.zeros(1, 32769, device="cuda"))
