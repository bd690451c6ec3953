"""Operands of more than 4 GiB: what offsets of 32 bits would reach wrongly is checked at the last rows."""
import pytest
import torch

from graphiler_amd import ops

pytestmark = pytest.mark.gpu
GIB = 1 << 30


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 40 * GIB:
        pytest.skip("needs 40 GiB of device memory")
    yield
    torch.cuda.empty_cache()


def test_norm_and_its_gradients():
    rows, cols = 2_200_003, 1024                         # 4.5 GB
    x = torch.randn(rows, cols, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(cols, device="cuda").bfloat16() + 0.5
    y, t = ops.rms_norm(x, w, x)
    y8, scales = ops.rms_norm_fp8(x, w)
    for part in (slice(0, 5), slice(rows - 5, rows)):    # rows do not depend on each other: the same bits
        a, b = ops.rms_norm(x[part], w, x[part])
        assert torch.equal(y[part], a) and torch.equal(t[part], b)
        a8, s8 = ops.rms_norm_fp8(x[part], w)
        assert torch.equal(y8[part].view(torch.uint8), a8.view(torch.uint8))
        assert torch.equal(scales[part].view(torch.uint8), s8.view(torch.uint8))
    gx, _ = ops.rms_norm_backward(y, x, w)
    a, _ = ops.rms_norm_backward(y[-5:], x[-5:], w)
    assert torch.equal(gx[-5:], a)


def test_gated_and_its_gradients():
    rows, k, f = 560_001, 4096, 128                      # 4.6 GB
    x = torch.randn(rows, k, device="cuda", dtype=torch.bfloat16)
    wg, wu = (torch.randn(k, f, device="cuda").bfloat16() / 64 for _ in range(2))
    h = ops.gated_linear(x, wg, wu)
    few = torch.cat([torch.arange(100), torch.arange(rows - 100, rows)]).cuda()
    # the same products and the same order along k, whatever the tile
    assert torch.equal(h[few], ops.gated_linear(x[few], wg, wu))
    gh = torch.zeros(rows, f, device="cuda", dtype=torch.bfloat16)
    gh[few] = torch.randn(200, f, device="cuda").bfloat16()
    gx, gg, gu = ops.gated_linear_backward(gh, x, wg, wu)
    assert not gx[100:-100].any()
    x64, gh64, wg64, wu64 = (t.double() for t in (x[few], gh[few], wg, wu))
    g, u = x64 @ wg64, x64 @ wu64
    s = torch.sigmoid(g)
    dg, du = gh64 * u * s * (1 + g * (1 - s)), gh64 * g * s
    # The result is rounded to bf16, 2^-8 of it, and dg and du are, 2^-8 of each.  Sums in fp32 are off by
    # up to their length times 2^-24 of their terms' sizes: g and u, whose errors reach dg and du by slopes of
    # at most 1.1 (silu) and 0.5 (its slope), and the sums of the results (of 256 or 200 terms that are not 0).
    eg, eu = (k * 2.0 ** -24 * (x64.abs() @ w.abs()) for w in (wg64, wu64))
    ddg = 2.0 ** -8 * dg.abs() + gh64.abs() * (0.5 * u.abs() * eg + 1.1 * eu)
    ddu = 2.0 ** -8 * du.abs() + 1.1 * gh64.abs() * eg
    for got, terms in ((gx[few], [(dg, wg64.t(), ddg), (du, wu64.t(), ddu)]), (gg, [(dg, x64.t(), ddg)]),
                       (gu, [(du, x64.t(), ddu)])):
        def product(a, b):
            return a @ b if len(terms) == 2 else b @ a
        want = sum(product(a, b) for a, b, _ in terms)
        room = sum(product(d + 256 * 2.0 ** -24 * a.abs(), b.abs()) for a, b, d in terms)
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * room).all()


def test_products_of_8_bits():
    rows, k, m = 560_001, 8192, 64                       # 4.6 GB
    x8 = torch.randint(0, 120, (rows, k), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    xs = torch.full((rows, k // 128), 127, device="cuda", dtype=torch.uint8)
    xs[-3:] = 124
    xs = xs.view(torch.float8_e8m0fnu)
    w8, ws = ops.quantize_weight_fp8(torch.randn(k, m, device="cuda"))
    y = ops.linear_fp8(x8, xs, w8, ws)
    for part in (slice(0, 200), slice(rows - 200, rows)):
        assert torch.equal(y[part], ops.linear_fp8(x8[part], xs[part], w8, ws))


def test_one_tensor_in_two_places():
    x = torch.randn(70, 96, device="cuda", requires_grad=True)
    w = (torch.randn(96, 40, device="cuda") / 10).requires_grad_()
    n = torch.rand(96, device="cuda").requires_grad_()
    y, t = ops.rms_norm(x, n, x)
    h = ops.gated_linear(y + t, w, w)
    gx, gw, gn = torch.autograd.grad(h, (x, w, n), torch.ones_like(h))
    x64, w64, n64 = (v.detach().double().requires_grad_() for v in (x, w, n))
    t64 = 2 * x64
    y64 = t64 / torch.sqrt((t64 * t64).mean(1, keepdim=True) + 1e-6) * n64
    g64 = (y64 + t64) @ w64
    h64 = torch.nn.functional.silu(g64) * g64
    want = torch.autograd.grad(h64, (x64, w64, n64), torch.ones_like(h64))
    # sums of at most 96 terms in fp32 (2^-24 a step), four of them one behind the other, relative to the largest
    for got, ref in zip((gx, gw, gn), want):
        assert (got.double() - ref).abs().max() <= 4 * 96 * 2.0 ** -24 * ref.abs().max()
