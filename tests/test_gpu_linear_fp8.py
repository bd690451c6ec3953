"""Products of 8-bit rows with block scales, plain and gated, against float64.

Bounds.  The matrix instruction adds eight products at a time and drops what lies 2^-13 below the
largest of them: at most 7 * 2^-13 < 2^-10 of their sizes' sum; K / 8 additions in fp32 follow.
Operands of few bits whose products and sums are whole numbers below 2^12 lose nothing.
"""
import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import capi, ops
from graphiler_amd.hipgraph import Graphed

pytestmark = pytest.mark.gpu


def wide(values, scales, rows_each):
    s = torch.exp2(scales.view(torch.uint8).double() - 127)
    s = s.repeat_interleave(rows_each, 0)[:values.shape[0]].repeat_interleave(128, 1)
    return values.double() * s


def make(seed, rows, k, m, pair=False, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen) * torch.exp(spread * torch.randn(k, generator=gen))
    ws = [torch.randn(k, m, generator=gen) / k ** 0.5 * torch.exp(spread * torch.randn(1, m, generator=gen))
          for _ in range(2 if pair else 1)]
    return ops.quantize_fp8(x.cuda()), [ops.quantize_weight_fp8(w.cuda()) for w in ws]


def bound(x, w, k):
    return (2.0 ** -10 + (k / 8 + 8) * 2.0 ** -24) * (x.abs() @ w.abs().t())


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, limit):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    worst = (err / (limit + 1e-30)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 4096, 300), (2, 200, 130), (3, 128, 4), (15, 500, 33), (16, 1000, 127),
          (17, 256, 128), (31, 128, 129), (33, 640, 257), (64, 384, 64), (100, 130, 1000), (128, 256, 128),
          (129, 1024, 66), (300, 128, 300), (5, 8192, 70), (32, 2048, 512)]
LARGE = [(3600, 256, 3600), (256 * 15, 384, 256 * 13)]


def check(rows, k, m, out_dtype):
    (x8, xs), [(w8, ws)] = make(rows + k + m, rows, k, m)
    y = ops.linear_fp8(x8, xs, w8, ws, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    x, w = wide(x8, xs, 1), wide(w8, ws, 128)
    want = x @ w.t()
    limit = bound(x, w, x.shape[1])
    within(y, want, limit + half_step(out_dtype) * (want.abs() + limit))
    if want.numel() > 64:
        off = (y.double() - want).norm() / want.norm()
        assert off <= half_step(out_dtype) + 2.0 ** -11, off


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k,m", SHAPES)
def test_against_float64(rows, k, m, out_dtype):
    check(rows, k, m, out_dtype)


@pytest.mark.parametrize("rows,k,m", LARGE)
def test_large_tiles(rows, k, m):
    check(rows, k, m, torch.bfloat16)


@pytest.mark.parametrize("rows,k,m", SHAPES + LARGE)
def test_whole_numbers_are_exact(rows, k, m):
    """Whole numbers up to 4 with a power of two each block, any eight products within 2^12 of each
    other: the sums of a block are exact, and so are all sums where the scales of a row agree."""
    gen = torch.Generator().manual_seed(k)
    kp = -(-k // 128) * 128
    x = torch.randint(-4, 5, (rows, kp), generator=gen).float()
    w = torch.randint(-4, 5, (m, kp), generator=gen).float()
    ex = torch.randint(-9, 9, (rows, 1), generator=gen).expand(rows, kp // 128).contiguous()
    ew = torch.randint(-9, 9, (-(-m // 128), 1), generator=gen).expand(-1, kp // 128).contiguous()
    # blocks may still differ where the sums stay small: the second block of a row is doubled
    if kp >= 256:
        ex[:, 1] += 1
    x8, w8 = x.to(torch.float8_e4m3fn).cuda(), w.to(torch.float8_e4m3fn).cuda()
    xs, ws = ((e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).cuda() for e in (ex, ew))
    y = ops.linear_fp8(x8, xs, w8, ws, out_dtype=torch.float32)
    assert torch.equal(y.double(), wide(x8, xs, 1) @ wide(w8, ws, 128).t())


@pytest.mark.parametrize("rows,k,m", [(70, 4224, 130), (70, 8192, 130), (70, 8320, 130), (100, 32768, 96), (2300, 8192, 2100),
                                      (2300, 8320, 2100), (3900, 8320, 3900)])
def test_many_blocks(rows, k, m):
    """Around the numbers of blocks that change what a tile keeps: whole numbers, so that all sums are exact (below
    2^24 of the smallest), and of the gated form one rounding of a product of exact numbers."""
    gen = torch.Generator().manual_seed(k)
    x = torch.randint(-4, 5, (rows, k), generator=gen).to(torch.float8_e4m3fn).cuda()
    wg, wu = (torch.randint(-4, 5, (m, k), generator=gen).to(torch.float8_e4m3fn).cuda() for _ in range(2))
    ex = torch.randint(-9, 9, (rows, 1), generator=gen).expand(rows, k // 128).contiguous()
    ex[:, -1] += 1                                       # the last block's scale is its own
    xs = (ex + 127).to(torch.uint8).view(torch.float8_e8m0fnu).cuda()
    ws = torch.full((-(-m // 128), k // 128), 125, dtype=torch.uint8).view(torch.float8_e8m0fnu).cuda()
    g, u = (wide(x, xs, 1) @ wide(w, ws, 128).t() for w in (wg, wu))
    assert torch.equal(ops.linear_fp8(x, xs, wg, ws, out_dtype=torch.float32).double(), g)
    h = ops.gated_linear_fp8(x, xs, wg, ws, wu, ws, activation="relu", out_dtype=torch.float32)
    assert torch.equal(h, torch.relu(g).float() * u.float())


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,f", [(1, 256, 512), (3, 128, 5), (17, 300, 127), (130, 256, 129), (70, 640, 1000),
                                      (3600, 128, 1800)])
def test_gated_against_float64(rows, k, f, act, out_dtype):
    if rows > 1000 and act != "silu":
        pytest.skip("one activation at the large size")
    (x8, xs), [(g8, gs), (u8, us)] = make(rows + f, rows, k, f, pair=True, spread=0.5)
    h = ops.gated_linear_fp8(x8, xs, g8, gs, u8, us, activation=act, out_dtype=out_dtype)
    x, wg, wu = wide(x8, xs, 1), wide(g8, gs, 128), wide(u8, us, 128)
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = bound(x, wg, x.shape[1]), bound(x, wu, x.shape[1])
    a = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[act](g)
    want = a * u
    limit = 1.13 * eg * (u.abs() + eu) + a.abs() * eu + (g.abs() + 8) * 2.0 ** -22 * (g * u).abs()
    within(h, want, limit + half_step(out_dtype) * (want.abs() + limit))
    if want.numel() > 64:
        off = (h.double() - want).norm() / want.norm()
        assert off <= half_step(out_dtype) + 2.0 ** -10, off


def test_nan_reaches_its_row_and_column_only():
    (x8, xs), [(w8, ws)] = make(3, 40, 256, 70)
    clean = ops.linear_fp8(x8, xs, w8, ws)
    x8.view(torch.uint8)[7, 200] = 0x7f                     # NaN in e4m3
    w8.view(torch.uint8)[11, 3] = 0xff
    y = ops.linear_fp8(x8, xs, w8, ws)
    assert bool(torch.isnan(y[7]).all()) and bool(torch.isnan(y[:, 11]).all())
    keep_r, keep_c = [i for i in range(40) if i != 7], [i for i in range(70) if i != 11]
    assert torch.equal(y[keep_r][:, keep_c], clean[keep_r][:, keep_c])
    (x8, xs), _ = make(3, 40, 256, 70)
    xs.view(torch.uint8)[5, 1] = 255                       # NaN among the scales
    y = ops.linear_fp8(x8, xs, w8, ws)
    assert bool(torch.isnan(y[5]).all())


@pytest.mark.parametrize("rows", [1, 40, 130])
def test_values_behind_the_results_are_left(rows):
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    for m in (5, 64, 70):
        (x8, xs), [(w8, ws)] = make(3, rows, 256, m)
        y = torch.full((rows * m + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        assert lib.ga_linear_fp8(x8.data_ptr(), xs.data_ptr(), w8.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, 256,
                                 m, capi.GA_BF16, stream) == 0
        assert bool((y[rows * m:] == 7).all())
        assert torch.equal(y[:rows * m].view(rows, m), ops.linear_fp8(x8, xs, w8, ws))


def test_no_rows_and_recorded_graphs():
    (x8, xs), [(w8, ws), (u8, us)] = make(4, 33, 256, 200, pair=True)
    assert ops.linear_fp8(x8[:0], xs[:0], w8, ws).shape == (0, 200)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(33, 256, generator=gen, device="cuda").bfloat16()
    norm = torch.ones(256, device="cuda").bfloat16()

    def step():
        y8, s = ops.rms_norm_fp8(x, norm)
        h = ops.gated_linear_fp8(y8, s, w8, ws, u8, us)
        return ops.linear_fp8(*ops.quantize_fp8(h), *down)

    down = ops.quantize_weight_fp8(torch.randn(200, 256, generator=gen, device="cuda"))
    g = Graphed(step)
    for _ in range(4):
        x.normal_(generator=gen)
        got = g().clone()
        assert torch.equal(got, step())
