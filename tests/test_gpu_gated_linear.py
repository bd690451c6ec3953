"""The gated half of a feed-forward block and its gradients, against float64.

Bounds.  A product of the kernel leaves out less than 2^-22 of every product of fp32 values (none of
bf16 ones) and adds n = K (fp32: 6 K) terms in fp32: it is off by at most (2^-22 + n 2^-24) sum |x||w|.
The activations use the hardware's exponential, off by (|g| + 8) 2^-22 at most.  Rounding to the type of the
result adds half a step of it.  dg and du are rounded to bf16 in bf16 (half a step each), which
reaches the gradients through the sizes of their products.
"""
import math

import pytest
import torch

from graphiler_amd import capi, ops
from graphiler_amd.hipgraph import Graphed

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
ACTS = ["silu", "gelu", "relu"]


def act64(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return torch.relu(g)


def slope64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return s * (1 + g * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return (g > 0).double()


def make(seed, rows, k, f, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen)
    wg, wu = (1.5 * torch.randn(k, f, generator=gen) / math.sqrt(k) for _ in range(2))
    gh = 0.1 * torch.randn(rows, f, generator=gen)
    return tuple(t.to(dtype).cuda() for t in (x, wg, wu, gh))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def product_bound(a, b, dtype, n=None):
    """Of a @ b formed by the kernel: (2^-22 + n 2^-24) |a| @ |b|."""
    n = (a.shape[1] if n is None else n) * (6 if dtype == torch.float32 else 1)
    return ((2.0 ** -22 if dtype == torch.float32 else 0) + (n + 4) * 2.0 ** -24) * (a.abs() @ b.abs())


def within(got, want, bound):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    worst = (err / (bound + 1e-30)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


SHAPES = [(1, 1, 1), (1, 8, 8), (2, 64, 64), (3, 7, 5), (16, 65, 66), (17, 128, 130), (33, 72, 4), (31, 300, 97),
          (64, 256, 64), (65, 100, 341), (127, 63, 63), (128, 64, 128), (129, 200, 257), (300, 40, 700),
          (1, 1024, 512), (5, 1000, 1003), (32, 512, 96), (257, 129, 72)]
# enough tiles for the workgroups of eight wavefronts
LARGE = [(3600, 72, 1800), (256 * 15, 136, 128 * 13)]


def check_forward(rows, k, f, dtype, act):
    x, wg, wu, _ = make(rows + k + f, rows, k, f, dtype)
    h = ops.gated_linear(x, wg, wu, act)
    assert h.dtype == dtype
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg, x @ wu
    eg, eu = product_bound(x, wg, dtype), product_bound(x, wu, dtype)
    want = act64(act, g) * u
    # |act'| < 1.13; gelu's error function cancels for negative g: 2^-22 of g itself
    bound = 1.13 * eg * (u.abs() + eu) + act64(act, g).abs() * eu + \
        (g.abs() + 8) * 2.0 ** -22 * (want.abs() + (g * u).abs() * (act == "gelu"))
    within(h, want, bound + half_step(dtype) * (want.abs() + bound))
    # far closer than the bound as a whole: fp32 sums of random signs
    off = (h.double() - want).norm() / want.norm()
    assert off <= half_step(dtype) + 2.0 ** -21, off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", SHAPES)
def test_forward_against_float64(rows, k, f, dtype):
    check_forward(rows, k, f, dtype, "silu")


# fp32: tiles of 32 and of 64 rows on the fp32 instruction, ends in k, rows and columns, one step and several;
# then few columns; then pieces in tiles of 64 and of 128 rows
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,k,f", [(50, 63, 97), (70, 64, 128), (33, 130, 31), (2708, 65, 341), (3001, 1, 353), (2720, 256, 352),
                                      (9001, 33, 96), (2048, 300, 704), (3000, 72, 1000)])
def test_fp32_tiles(rows, k, f, act):
    check_forward(rows, k, f, torch.float32, act)


@pytest.mark.parametrize("rows", [20, 2708])
def test_fp32_infinities_and_small_values_of_few_tiles(rows):
    x = torch.zeros(rows, 96)
    x[0, 3], x[1, 4], x[rows - 1] = math.inf, 1e-36, 1.0
    w = torch.ones(96, 341)
    got = ops.gated_linear(x.cuda(), w.cuda(), w.cuda(), "relu").cpu()
    assert (got[0] == math.inf).all() and (got[rows - 1] == 96 * 96).all()
    got = ops.gated_linear(x.cuda(), w.cuda(), 1e36 * w.cuda(), "relu").cpu()
    # 1e-36 times (1e-36 times 1e36): two roundings of operands, two of products, one of the bound
    assert ((got[1].double() / 1e-36 - 1.0).abs() <= 5 * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,k,f", [(4, 96, 80), (150, 75, 133)])
def test_activations(rows, k, f, dtype, act):
    check_forward(rows, k, f, dtype, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", LARGE)
def test_large_tiles(rows, k, f, dtype):
    check_forward(rows, k, f, dtype, "silu")


def check_backward(rows, k, f, dtype, act):
    x, wg, wu, gh = make(rows + k * f, rows, k, f, dtype)
    got = ops.gated_linear_backward(gh, x, wg, wu, act)
    assert [t.shape for t in got] == [x.shape, wg.shape, wu.shape] and all(t.dtype == dtype for t in got)
    x, wg, wu, gh = x.double(), wg.double(), wu.double(), gh.double()
    g, u = x @ wg, x @ wu
    eg, eu = product_bound(x, wg, dtype), product_bound(x, wu, dtype)
    dg, du = gh * u * slope64(act, g), gh * act64(act, g)
    soft = (g.abs() + 8) * 2.0 ** -22
    # |act''| < 1 away from relu's corner; there the slope may be either where |g| is within its error
    corner = (g.abs() <= eg).double() if act == "relu" else 0.0
    rounds = half_step(dtype) if dtype == torch.bfloat16 else 2.0 ** -22
    e_dg = gh.abs() * ((u.abs() + eu) * (eg * (act != "relu") + soft * 1.2 + corner) + 1.13 * eu)
    e_du = gh.abs() * (1.13 * eg + soft * (g.abs() + eg))
    e_dg, e_du = e_dg + rounds * (dg.abs() + e_dg), e_du + rounds * (du.abs() + e_du)
    sums = (2.0 ** -22 if dtype == torch.float32 else 0) + 2.0 ** -24 * 16
    many = 6 if dtype == torch.float32 else 1

    def weight(d, e):
        size = x.t().abs() @ (d.abs() + e)
        return x.t() @ d, x.t().abs() @ e + (sums + many * rows * 2.0 ** -24) * size

    wx = dg @ wg.t() + du @ wu.t()
    size = (dg.abs() + e_dg) @ wg.t().abs() + (du.abs() + e_du) @ wu.t().abs()
    bx = e_dg @ wg.t().abs() + e_du @ wu.t().abs() + (sums + 2 * many * f * 2.0 ** -24) * size
    for name, mine, (want, bound) in zip(("x", "gate", "up"), got, ((wx, bx), weight(dg, e_dg), weight(du, e_du))):
        within(mine, want, bound + half_step(dtype) * (want.abs() + bound))
        if want.numel() > 64 and act != "relu":
            off = (mine.double() - want).norm() / want.norm()
            # two roundings of bf16 side by side; fp32: sums of random signs
            assert off <= (2 * half_step(dtype) if dtype == torch.bfloat16 else 2.0 ** -20), (name, off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", SHAPES)
def test_gradients_against_float64(rows, k, f, dtype):
    check_backward(rows, k, f, dtype, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,k,f", [(40, 96, 80), (150, 75, 133)])
def test_gradients_of_activations(rows, k, f, dtype, act):
    check_backward(rows, k, f, dtype, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(3600, 72, 1800), (700, 1800, 1900), (5000, 136, 40)])
def test_gradients_with_large_tiles_and_long_sums(rows, k, f, dtype):
    check_backward(rows, k, f, dtype, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(8192, 1280, 40), (70, 2048, 2600)])
def test_gradients_of_rows_and_of_weights_with_large_tiles(rows, k, f, dtype):
    check_backward(rows, k, f, dtype, "silu")


def test_gradients_against_differences():
    x, wg, wu, gh = make(2, 9, 40, 24, torch.float32)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    (ops.gated_linear(*leaves) * gh).sum().backward()
    gen = torch.Generator(device="cuda").manual_seed(3)

    def value(at):
        g, u = at[0].double() @ at[1].double(), at[0].double() @ at[2].double()
        return (act64("silu", g) * u * gh.double()).sum().item()

    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=gen, device="cuda")
        at = [t.detach() for t in leaves]
        up, down = list(at), list(at)
        up[i], down[i] = at[i].double() + 2.0 ** -10 * d, at[i].double() - 2.0 ** -10 * d
        slope = (value(up) - value(down)) * 2.0 ** 9
        assert abs(slope - (leaf.grad * d).sum().item()) <= 2.0 ** -12 * (leaf.grad.abs() * d.abs()).sum().item() + 1e-6


def test_no_rows():
    x, wg, wu, gh = make(1, 4, 24, 16, torch.bfloat16)
    assert ops.gated_linear(x[:0], wg, wu).shape == (0, 16)
    gx, gg, gu = ops.gated_linear_backward(gh[:0], x[:0], wg, wu)
    assert gx.shape == (0, 24) and bool((gg == 0).all()) and bool((gu == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [6, 200])
def test_a_row_that_is_not_finite_stays_alone(dtype, rows):
    x, wg, wu, _ = make(8, rows, 100, 90, dtype)
    clean = ops.gated_linear(x, wg, wu)
    x[2, 5], x[4, 99] = float("nan"), float("inf")
    h = ops.gated_linear(x, wg, wu)
    keep = [i for i in range(rows) if i not in (2, 4)]
    assert torch.equal(h[keep], clean[keep])
    assert bool(torch.isnan(h[2]).all())
    assert not bool(torch.isfinite(h[4]).any()) or dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(3, 64, 40), (130, 65, 67), (64, 64, 66)])
def test_values_behind_the_results_are_left(rows, k, f, dtype):
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    dt = capi.GA_F32 if dtype == torch.float32 else capi.GA_BF16
    x, wg, wu, gh = make(5, rows, k, f, dtype)
    n = lib.ga_gated_linear_backward_workspace_bytes(rows, k, f, dt)
    ws = torch.full((n + 256,), 171, dtype=torch.uint8, device="cuda")
    sizes = [rows * f, rows * k, k * f, k * f]
    h, gx, gg, gu = (torch.full((m + 64,), 7.0, dtype=dtype, device="cuda") for m in sizes)
    assert lib.ga_gated_linear(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), rows, k, f, 0, dt,
                               ws.data_ptr(), n, stream) == 0
    assert lib.ga_gated_linear_backward(gh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gx.data_ptr(),
                                        gg.data_ptr(), gu.data_ptr(), rows, k, f, 0, dt, ws.data_ptr(), n, stream) == 0
    for t, m in zip((h, gx, gg, gu), sizes):
        assert bool((t[m:] == 7).all()) and not bool((t[:m] == 7).all())
    assert bool((ws[n:] == 171).all())
    # whatever the workspace held before
    ws.fill_(255)
    again = torch.empty_like(gg)
    assert lib.ga_gated_linear_backward(gh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gx.data_ptr(),
                                        again.data_ptr(), gu.data_ptr(), rows, k, f, 0, dt, ws.data_ptr(), n, stream) == 0
    assert torch.equal(again[:k * f], gg[:k * f])


@pytest.mark.parametrize("rows,k,f,dtype", [(2, 256, 512, torch.bfloat16), (300, 130, 200, torch.float32)])
def test_recorded_graphs_replay(rows, k, f, dtype):
    x, wg, wu, gh = make(6, rows, k, f, dtype)

    def step():
        return (ops.gated_linear(x, wg, wu), *ops.gated_linear_backward(gh, x, wg, wu))

    g = Graphed(step)
    for seed in range(4):
        x.copy_(make(60 + seed, rows, k, f, dtype)[0])
        got = [t.clone() for t in g()]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream_and_repeats_are_the_same():
    x, wg, wu, gh = make(12, 500, 200, 300, torch.bfloat16)
    want = (ops.gated_linear(x, wg, wu), *ops.gated_linear_backward(gh, x, wg, wu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ops.gated_linear(x, wg, wu), *ops.gated_linear_backward(gh, x, wg, wu))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gradients_arrive_through_views():
    x, wg, wu, _ = make(13, 20, 32, 48, torch.float32)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    ops.gated_linear(*leaves).sum().backward()                # an expanded gradient
    wide = [t.detach().double().requires_grad_() for t in leaves]
    (act64("silu", wide[0] @ wide[1]) * (wide[0] @ wide[2])).sum().backward()
    for a, b in zip(leaves, wide):
        assert (a.grad.double() - b.grad).norm() <= 2.0 ** -19 * b.grad.norm()


def test_recording_with_gradients_is_refused():
    x, wg, wu, _ = make(13, 20, 32, 48, torch.float32)
    wg.requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            ops.gated_linear(x, wg, wu)
        with torch.no_grad():
            h = ops.gated_linear(x, wg, wu)
    graph.replay()
    assert torch.equal(h, ops.gated_linear(x, wg.detach(), wu))
