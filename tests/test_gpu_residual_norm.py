"""Root-mean-square norm with the residual's addition, its gradients, and rows cut to 8 bits,
against the same expressions in float64.

Bounds: a value stored in a type is off by at most half a step of it (eps / 2, relative).  In fp32 a
lane adds up to 64 squares one after the other, then eight levels of pairs: the mean square is off by
at most 72 * 2^-24, its root by half of that, and four more roundings follow: 42 * 2^-24.
"""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import capi, ops
from graphiler_amd.hipgraph import Graphed

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
STEPS = 42 * 2.0 ** -24
EPS = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(seed, rows, cols, dtype, residual=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen))
    r = torch.randn(rows, cols, generator=gen) if residual else None
    w = 1 + 0.3 * torch.randn(cols, generator=gen)
    return tuple(None if t is None else t.to(dtype).cuda() for t in (x, r, w))


def exact(x, r, w, eps=EPS):
    t = x.double() if r is None else x.double() + r.double()
    return t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * w.double(), t


def within(got, want, bound):
    err = (got.double() - want).abs()
    worst = (err / (bound + 1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


SHAPES = [(1, 1), (1, 16), (3, 7), (2, 8), (5, 100), (17, 128), (9, 129), (33, 256), (4, 257), (70, 500),
          (6, 512), (3, 513), (5, 1000), (4, 1024), (3, 1025), (2, 2047), (3, 2048), (2, 4090), (2, 4096),
          (3, 5001), (2, 8192), (2, 8193), (1, 16384), (0, 64), (4097, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm_against_float64(rows, cols, dtype):
    for residual in (True, False):
        x, r, w = make(rows + cols, rows, cols, dtype, residual)
        got = ops.rms_norm(x, w, r, eps=EPS)
        y, t = got if residual else (got, None)
        want, total = exact(x, r, w)
        assert y.dtype == dtype and y.shape == x.shape
        # the sum is rounded to fp32 first: one more step where it is small beside its terms
        slip = 2.0 ** -24 * total.abs()
        within(y, want, want.abs() * (half_step(dtype) * (1 + STEPS) + STEPS))
        if residual:
            within(t, total, total.abs() * half_step(dtype) + slip)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_8bit_rows(rows, cols, dtype):
    x, r, w = make(rows + 2 * cols, rows, cols, dtype)
    y8, scales, t = ops.rms_norm_fp8(x, w, r, eps=EPS)
    blocks = -(-cols // 128)
    assert y8.shape == (rows, 128 * blocks) and scales.shape == (rows, blocks)
    assert y8.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    want, total = exact(x, r, w)
    assert torch.equal(t, ops.rms_norm(x, w, r, eps=EPS)[1])
    s = torch.exp2(scales.view(torch.uint8).double() - 127)
    padded = F.pad(want, (0, 128 * blocks - cols)).view(rows, blocks, 128)
    top = padded.abs().amax(2)
    # the smallest power of two, up to what the norm's own rounding may move a maximum across a border
    assert bool((top <= 448 * s * (1 + STEPS)).all())
    assert bool(((top > 224 * s * (1 - STEPS)) | (top == 0)).all())
    held = y8.double().view(rows, blocks, 128) * s.unsqueeze(2)
    # half a step of a normal e4m3 value, half the step of its subnormals
    within(held, padded, padded.abs() * (2.0 ** -4 + STEPS) + s.unsqueeze(2) * 2.0 ** -10)
    assert bool((held.reshape(rows, 128 * blocks)[:, cols:] == 0).all())


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_8bit_norm_is_the_norm_cut_to_8_bits(rows, cols):
    x, r, w = make(7, rows, cols, torch.float32)
    y8, scales, _ = ops.rms_norm_fp8(x, w, r)
    cut8, cut_scales = ops.quantize_fp8(ops.rms_norm(x, w, r)[0])
    assert torch.equal(y8.view(torch.uint8), cut8.view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), cut_scales.view(torch.uint8))


def plain_cut(x):
    """Rows cut to 8 bits on the host, by the definition."""
    x = x.float().cpu().numpy()
    rows, cols = x.shape
    blocks = -(-cols // 128)
    padded = np.zeros((rows, blocks * 128), np.float32)
    padded[:, :cols] = x
    b = padded.reshape(rows, blocks, 128)
    top = np.where(np.isfinite(b), np.abs(b), 0).max(2)
    e = np.zeros(top.shape, np.int64)
    live = top > 0
    e[live] = np.ceil(np.log2(top[live].astype(np.float64) / 448)).astype(np.int64)
    e = np.clip(e, -126, 126)
    # the logarithm is exact to far below the distance of two floats: check the borders themselves
    assert np.all(top <= 448 * 2.0 ** e) and np.all((top > 224 * 2.0 ** e) | (e == -126) | ~live)
    v = b.astype(np.float64) * (2.0 ** -e.astype(np.float64))[:, :, None]
    v = np.where(np.isfinite(v), v, np.nan)
    return torch.from_numpy(v.astype(np.float32)).to(torch.float8_e4m3fn).view(rows, -1), \
        torch.from_numpy((e + 127).astype(np.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (5, 200), (33, 1000), (2, 4096), (1, 16384)])
def test_quantize_bit_for_bit(rows, cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(6 * torch.randn(rows, cols, generator=gen))
    x[0, 0] = 448.0                                       # a border: scale 1, the largest value
    x = x.to(dtype)
    x8, scales = ops.quantize_fp8(x.cuda())
    want8, want_scales = plain_cut(x)
    assert torch.equal(scales.view(torch.uint8).cpu(), want_scales)
    assert torch.equal(x8.cpu().view(torch.uint8), want8.view(torch.uint8))


def test_quantize_borders():
    x = torch.zeros(10, 128)
    x[1] = 1e-45                                          # below the smallest scale
    x[2, 3] = 448.0
    x[3, 3] = float(np.nextafter(np.float32(448), np.float32(500)))
    x[4, 5] = 3.0e38
    x[5, 5], x[5, 6], x[5, 7] = float("inf"), 2.0, float("nan")
    x[6] = float("-inf")
    x[7, 0], x[7, 1] = -448.0 * 2.0 ** -126, 2.0 ** -126
    x[8, 0], x[8, 1], x[8, 2] = 256.0, 2.0 ** -7 + 2.0 ** -10, 2.0 ** -10     # ties among the subnormals
    x[9, 0], x[9, 1] = 17.0 * 16, 19.0 * 16                                # ties go to even
    x8, scales = ops.quantize_fp8(x.cuda())
    want8, want_scales = plain_cut(x)
    assert torch.equal(scales.view(torch.uint8).cpu(), want_scales)
    got, want = x8.cpu().float(), want8.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert want_scales[0, 0] == 127 and want_scales[2, 0] == 127 and want_scales[3, 0] == 128


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,m", [(1, 1), (128, 128), (130, 127), (300, 257), (64, 1000)])
def test_quantize_weight_bit_for_bit(k, m, dtype):
    gen = torch.Generator().manual_seed(k)
    w = (torch.randn(k, m, generator=gen) * torch.exp(2 * torch.randn(1, m, generator=gen))).to(dtype)
    w8, scales = ops.quantize_weight_fp8(w.cuda())
    kb, mb = -(-k // 128), -(-m // 128)
    assert w8.shape == (m, kb * 128) and scales.shape == (mb, kb)
    t = F.pad(w.float().t(), (0, kb * 128 - k, 0, mb * 128 - m)).contiguous()
    tiles = t.view(mb, 128, kb, 128).permute(0, 2, 1, 3).reshape(mb * kb, 128 * 128)
    top = tiles.abs().amax(1).double()
    e = torch.ceil(torch.log2(top / 448)).clamp(-126, 126)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    assert torch.equal(scales.view(torch.uint8).cpu().double().view(-1), e + 127)
    v = (tiles.double() * torch.exp2(-e).unsqueeze(1)).float().view(mb, kb, 128, 128).permute(0, 2, 1, 3)
    want = v.reshape(mb * 128, kb * 128)[:m].to(torch.float8_e4m3fn)
    assert torch.equal(w8.cpu().view(torch.uint8), want.contiguous().view(torch.uint8))


GRAD_SHAPES = [(1, 1), (3, 7), (17, 128), (40, 129), (33, 256), (70, 500), (5, 1000), (3, 2048), (9, 4090),
               (2, 8192), (2, 16384), (5000, 40), (3000, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", GRAD_SHAPES)
def test_gradients_against_float64(rows, cols, dtype):
    x, r, w = make(rows * 3 + cols, rows, cols, dtype)
    gen = torch.Generator().manual_seed(5)
    gy = (0.1 * torch.randn(rows, cols, generator=gen)).to(dtype).cuda()
    for gt in (r, None):
        gx, gw = ops.rms_norm_backward(gy, x, w, EPS, gt)
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y = x64 / torch.sqrt((x64 * x64).mean(1, keepdim=True) + EPS) * w64
        wx, ww = torch.autograd.grad(y, (x64, w64), gy.double())
        wx = wx if gt is None else wx + gt.double()
        t, g, v = x.double(), gy.double(), w.double()
        inv = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
        # a term is three or four roundings and powers of the root: each is off by at most 4 STEPS
        size = inv * (v * g).abs() + t.abs() * inv ** 3 * (t * v * g).abs().mean(1, keepdim=True)
        within(gx, wx, 4 * STEPS * size + (half_step(dtype) + 2.0 ** -24) * wx.abs())
        # sums over the rows: `rows` additions at most
        terms = (g * t * inv).abs().sum(0)
        within(gw, ww, (rows * 2.0 ** -24 + 2 * STEPS) * terms + half_step(dtype) * ww.abs())


def test_gradients_against_differences():
    x, r, w = make(3, 6, 200, torch.float32)
    x.requires_grad_(), r.requires_grad_(), w.requires_grad_()
    gen = torch.Generator(device="cuda").manual_seed(1)
    a, b = (torch.randn(6, 200, generator=gen, device="cuda") for _ in range(2))
    y, t = ops.rms_norm(x, w, r)
    ((y * a).sum() + (t * b).sum()).backward()

    def value(dx, dr, dw):
        y, t = exact((x + dx).detach(), (r + dr).detach(), (w + dw).detach())
        return ((y * a).sum() + (t * b).sum()).item()

    for i, leaf in enumerate((x, r, w)):
        d = torch.randn(leaf.shape, generator=gen, device="cuda")
        step = [torch.zeros_like(l) for l in (x, r, w)]
        step[i] = 2.0 ** -8 * d
        slope = (value(*step) - value(*(-s for s in step))) / 2.0 ** -7
        # central differences: h^2 / 6 of a third derivative of the size of the function
        assert abs(slope - (leaf.grad * d).sum().item()) <= 2.0 ** -9 * (leaf.grad.abs() * d.abs()).sum().item()


def test_autograd_of_parts():
    x, r, w = make(4, 5, 96, torch.float32)
    for used in ("y", "sum", "both"):
        leaves = [t.clone().requires_grad_() for t in (x, r, w)]
        y, t = ops.rms_norm(leaves[0], leaves[2], leaves[1])
        out = y.sum() if used == "y" else t.sum() if used == "sum" else y.sum() + 2 * t.sum()
        out.backward()
        wide = [l.detach().double().requires_grad_() for l in leaves]
        ye, te = exact(wide[0], wide[1], wide[2])
        (ye.sum() if used == "y" else te.sum() if used == "sum" else ye.sum() + 2 * te.sum()).backward()
        for got, want in zip(leaves, wide):
            if got.grad is None:
                assert want.grad is None or bool((want.grad == 0).all())
                continue
            assert torch.allclose(got.grad.double(), want.grad, rtol=2e-5, atol=2e-5)


def test_one_row_that_is_not_finite_stays_alone():
    x, r, w = make(9, 8, 300, torch.bfloat16)
    clean = ops.rms_norm(x, w, r)[0]
    x[3, 17], x[5, 0] = float("nan"), float("inf")
    y = ops.rms_norm(x, w, r)[0]
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep])
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[5, 0]))
    y8, scales, _ = ops.rms_norm_fp8(x, w, r)
    clean8 = ops.rms_norm_fp8(x[keep].contiguous(), w, r[keep].contiguous())[0]
    assert torch.equal(y8[keep].view(torch.uint8), clean8.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_are_left(dtype):
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    dt = capi.GA_F32 if dtype == torch.float32 else capi.GA_BF16
    for rows, cols in ((5, 200), (3, 129), (2, 3000), (7, 40)):
        x, r, w = make(1, rows, cols, dtype)
        y = torch.full((rows * cols + 64,), 7.0, dtype=dtype, device="cuda")
        t = torch.full((rows * cols + 64,), 7.0, dtype=dtype, device="cuda")
        assert lib.ga_rms_norm(x.data_ptr(), r.data_ptr(), w.data_ptr(), y.data_ptr(), t.data_ptr(), rows, cols,
                               EPS, dt, stream) == 0
        assert bool((y[rows * cols:] == 7).all()) and bool((t[rows * cols:] == 7).all())
        padded = -(-cols // 128) * 128
        y8 = torch.full((rows * padded + 64,), 9, dtype=torch.uint8, device="cuda")
        s = torch.full((rows * padded // 128 + 64,), 9, dtype=torch.uint8, device="cuda")
        assert lib.ga_rms_norm_fp8(x.data_ptr(), None, w.data_ptr(), y8.data_ptr(), s.data_ptr(), None, rows,
                                   cols, EPS, dt, stream) == 0
        assert bool((y8[rows * padded:] == 9).all()) and bool((s[rows * padded // 128:] == 9).all())


def test_in_place_sum_is_the_same():
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    x, r, w = make(2, 9, 700, torch.float32)
    y, t = ops.rms_norm(x, w, r)
    y2 = torch.empty_like(y)
    assert lib.ga_rms_norm(x.data_ptr(), r.data_ptr(), w.data_ptr(), y2.data_ptr(), r.data_ptr(), 9, 700, 1e-6,
                           capi.GA_F32, stream) == 0
    assert torch.equal(y, y2) and torch.equal(r, t)


def test_other_streams_and_recorded_graphs():
    x, r, w = make(11, 300, 512, torch.bfloat16)
    want = ops.rms_norm(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rms_norm(x, w, r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    def step():
        y, t = ops.rms_norm(x, w, r)
        gx, gw = ops.rms_norm_backward(y, t, w, 1e-6, r)
        return y, t, gx, gw

    g = Graphed(step)
    for k in range(4):
        x.copy_(make(20 + k, 300, 512, torch.bfloat16)[0])
        got = [a.clone() for a in g()]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_recording_with_gradients_is_refused():
    x, r, w = make(11, 8, 64, torch.float32)
    x.requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            ops.rms_norm(x, w, r)
        with torch.no_grad():
            y, _ = ops.rms_norm(x, w, r)
    graph.replay()
    assert torch.equal(y, ops.rms_norm(x.detach(), w, r)[0])
