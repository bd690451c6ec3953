"""Projections with bias, activation and residual against the definition in 64 bits.

Bounds, u = 2^-24 and r half a step of the tensors' type: a product of K terms is off by (K + 8) u + 2^-21 of the sum of
its terms' magnitudes (what fp32 products of pieces leave out is below 2^-22 of each); an activation passes
that on with a slope of at most 1.2 and is off by 2^-20 (|z| + 8) of |z| itself at most, its slope, whose own slope is at
most 1, by 2^-20 (|z| + 8) besides; dz is rounded by r as an operand where the tensors are bf16, results by r."""
import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
ACTS = {None: lambda z: z, "silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def operands(rows, k, m, dtype, bias, residual, seed=0):
    return (made((rows, k), dtype, seed), made((k, m), dtype, seed + 1, k ** -0.5), made((m,), dtype, seed + 2) if bias else None,
            made((rows, m), dtype, seed + 3) if residual else None)


def product_bound(a, b):
    return ((a.shape[1] + 8) * U + 2.0 ** -21) * (a.abs() @ b.abs())


def within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / tol)[bad].max()):.3g} times its bound"


def check_forward(rows, k, m, dtype, act, bias=True, residual=True, seed=0):
    x, w, b, r = operands(rows, k, m, dtype, bias, residual, seed)
    got = ops.linear_act(x, w, bias=b, activation=act, residual=r)
    xd, wd = x.double(), w.double()
    z = xd @ wd + (b.double() if bias else 0)
    off = product_bound(xd, wd) + 2 * U * z.abs()
    y = ACTS[act](z)
    off = 1.2 * off + (0 if act is None else 2.0 ** -20 * (z.abs() + 8) * z.abs())
    if residual:
        y = y + r.double()
    within(got, y, off + 2 * U * y.abs() + HALF_STEP[dtype] * y.abs() + 1e-37, "y")
    assert torch.equal(got, ops.linear_act(x, w, bias=b, activation=act, residual=r))


def check_backward(rows, k, m, dtype, act, bias=True, seed=0):
    x, w, b, _ = operands(rows, k, m, dtype, bias, False, seed)
    gy = made((rows, m), dtype, seed + 5, 0.1)
    got = ops.linear_act_backward(gy, x, w, bias=b, activation=act)
    xd, wd, gd = x.double(), w.double(), gy.double()
    r = HALF_STEP[dtype]
    z = (xd @ wd + (b.double() if bias else 0)).requires_grad_()
    if act is None:
        dz, off = gd, torch.zeros_like(gd)
    else:
        dz, = torch.autograd.grad(ACTS[act](z), z, gd)
        z = z.detach()
        z_off = product_bound(xd, wd) + 2 * U * z.abs()
        off = gd.abs() * (z_off + 2.0 ** -20 * (z.abs() + 8))
        if act == "relu":                     # next to 0 its slope may be either
            off = torch.where(z.abs() <= z_off, gd.abs(), 2 * U * gd.abs())
        off = off + (r if dtype == torch.bfloat16 else 4 * U) * (dz.abs() + off)
    want = (dz @ wd.t(), xd.t() @ dz, dz.sum(0))
    tol = (off @ wd.t().abs() + product_bound(dz, wd.t()), xd.t().abs() @ off + product_bound(xd.t(), dz),
           off.sum(0) + (rows + 8) * U * dz.abs().sum(0))
    for name, g, v, t in zip(("x", "weight", "bias"), got, want, tol):
        if g is None:
            assert name == "bias" and not bias
            continue
        within(g, v, t + r * (v.abs() + t) + 1e-37, "gradient of " + name)
    again = ops.linear_act_backward(gy, x, w, bias=b, activation=act)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, again))


SHAPES = [(1, 1, 1), (1, 1024, 512), (3, 100, 333), (8, 64, 64), (9, 130, 257), (16, 2048, 130), (17, 17, 17), (33, 64, 128),
          (64, 2048, 64), (100, 300, 700), (257, 129, 513), (1000, 512, 512), (2001, 72, 1000), (5000, 256, 96)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,m", SHAPES)
def test_forward(rows, k, m, dtype):
    for act in ACTS:
        check_forward(rows, k, m, dtype, act)
    check_forward(rows, k, m, dtype, None, bias=False, residual=False)
    check_forward(rows, k, m, dtype, "gelu", bias=False)
    check_forward(rows, k, m, dtype, "silu", residual=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,m", SHAPES)
def test_backward(rows, k, m, dtype):
    for act in ACTS:
        check_backward(rows, k, m, dtype, act)
    check_backward(rows, k, m, dtype, "gelu", bias=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [2048, 2000, 2004, 2047, 1290])
def test_the_largest_tiles(m, dtype):
    """More rows and columns than small tiles fill: 256 x 256 of bf16, taken as two products of 128 columns side by side."""
    rows = 9000 if dtype == torch.bfloat16 else 4100
    check_forward(rows, 192, m, dtype, "gelu")
    check_forward(rows, 70, m, dtype, None, bias=False)
    check_backward(rows, 192, m, dtype, "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_at_any_address_and_a_result_over_the_residual(dtype):
    for rows in (5, 40):
        x, w, b, r = operands(rows, 64, 96, dtype, True, True)
        apart = [torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (x, w, b, r)]
        want = ops.linear_act(x, w, bias=b, activation="gelu", residual=r)
        assert torch.equal(ops.linear_act(apart[0], apart[1], bias=apart[2], activation="gelu", residual=apart[3]), want)
        gy = made((rows, 96), dtype, 9)
        far = torch.empty(gy.numel() + 1, dtype=dtype, device=DEV)[1:].view(gy.shape).copy_(gy)
        for a, b2 in zip(ops.linear_act_backward(gy, x, w, bias=b, activation="gelu"),
                         ops.linear_act_backward(far, apart[0], apart[1], bias=apart[2], activation="gelu")):
            assert torch.equal(a, b2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,m", [(5, 64, 96), (40, 2048, 70), (700, 64, 256), (9000, 64, 512)])
def test_the_c_entry_writes_over_the_residual(rows, k, m, dtype):
    x, w, b, r = operands(rows, k, m, dtype, True, True)
    want = ops.linear_act(x, w, bias=b, activation="silu", residual=r)
    lib, dt = capi.load(), ops._DTYPES[dtype]
    n = lib.ga_linear_act_workspace_bytes(rows, k, m, dt)
    ws = torch.empty(n + 16, dtype=torch.uint8, device=DEV)
    assert lib.ga_linear_act(x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), r.data_ptr(), rows, k, m, capi.GA_GATE_SILU, dt,
                             ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(r, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows(dtype):
    x, w, b, r = operands(0, 64, 96, dtype, True, True)
    assert ops.linear_act(x, w, bias=b, activation="relu", residual=r).shape == (0, 96)
    gx, gw, gb = ops.linear_act_backward(made((0, 96), dtype, 1), x, w, bias=b, activation="relu")
    assert gx.shape == (0, 64) and not gw.any() and not gb.any() and gw.shape == w.shape and gb.shape == b.shape


def test_autograd():
    x, w, b, r = (t.requires_grad_() for t in operands(50, 40, 30, torch.float32, True, True))
    y = ops.linear_act(x, w, bias=b, activation="gelu", residual=r)
    gy = made((50, 30), torch.float32, 11)
    got = torch.autograd.grad(y, (x, w, b, r), gy)
    gx, gw, gb = ops.linear_act_backward(gy, x.detach(), w.detach(), bias=b.detach(), activation="gelu")
    assert all(torch.equal(a, b2) for a, b2 in zip(got, (gx, gw, gb, gy)))
    # against differences of the definition in 64 bits
    args = [t.detach().double() for t in (x, w, b, r)]
    f = lambda *a: (F.gelu(a[0] @ a[1] + a[2]) + a[3]).mul(gy.double()).sum()  # noqa: E731
    for i, g in enumerate(got):
        step = torch.randn_like(args[i])
        up, down = ([a + s * 1e-5 * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = (f(*up) - f(*down)) / 2e-5
        assert abs(slope - (g.double() * step).sum()) <= 1e-4 * (g.double() * step).abs().sum()
    only = torch.autograd.grad(ops.linear_act(x, w.detach(), bias=b.detach(), activation="gelu"), x, gy)[0]
    assert torch.equal(only, gx)
