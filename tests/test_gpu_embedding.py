"""Embedding rows and their table's gradient: the lookup bit by bit, the sums within what their length allows."""
import pytest
import torch

from graphiler_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BOTH = [torch.bfloat16, torch.float32]


def made(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def ids_of(n, rows, seed, bits=64, skew=1.0, pad=0.1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ids = (torch.rand(n, generator=gen, device=DEV).pow(skew) * rows).long().clamp(max=rows - 1)
    ids[torch.rand(n, generator=gen, device=DEV) < pad] = -1
    ids[torch.rand(n, generator=gen, device=DEV) < pad / 2] = rows + 5
    return ids if bits == 64 else ids.int()


def check(n, rows, cols, dtype, bits=64, skew=1.0, scale=1.7, pad=0.1):
    ids = ids_of(n, rows, n + rows, bits, skew, pad)
    table = made((rows, cols), dtype, 1)
    there = ((ids >= 0) & (ids < rows)).unsqueeze(1)
    safe = ids.long().clamp(0, rows - 1)
    factor = torch.tensor(scale, dtype=torch.float32, device=DEV)
    want = torch.where(there, table[safe].float() * factor, torch.zeros((), device=DEV)).to(dtype)
    assert torch.equal(ops.embedding(table, ids, scale=scale), want)
    gy = made((n, cols), dtype, 2)
    got = ops.embedding_backward(gy, ids, rows, scale=scale)
    sums = torch.zeros(rows, cols, dtype=torch.float64, device=DEV)
    mags, counts = torch.zeros_like(sums), torch.zeros(rows, 1, dtype=torch.float64, device=DEV)
    g = gy.double() * there
    sums.index_add_(0, safe, g)
    mags.index_add_(0, safe, g.abs())
    counts.index_add_(0, safe, there.double())
    s = float(factor)
    tol = ((counts + 8) * U * mags + HALF_STEP[dtype] * sums.abs()) * abs(s) * (1 + 1e-6) + 1e-37
    off = (got.double() - sums * s).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert torch.equal(got, ops.embedding_backward(gy, ids, rows, scale=scale))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("cols", [1, 7, 8, 64, 65, 100, 128, 256, 300, 512, 513, 1500])
def test_widths(cols, dtype):
    check(1000, 90, cols, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bits", [64, 32])
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 1000), (127, 1), (128, 1), (129, 1), (1000, 1), (1024, 8192), (1000, 65536), (1024, 65537), (1025, 300), (1024, 8193), (600, 40), (5000, 2), (257, 65), (20000, 7),
                                    (30000, 3000), (3000, 30000), (100000, 64)])
def test_counts(n, rows, bits, dtype):
    check(n, rows, 48, dtype, bits)
    check(n, rows, 520, dtype, bits, skew=4.0)


@pytest.mark.parametrize("dtype", BOTH)
def test_runs_that_begin_and_end_with_the_cuts(dtype):
    """Rows of exactly 128, 129, 256 and 257 places, one behind the other in every order."""
    for counts in ([128] * 4, [129, 127, 256, 1], [257, 128, 127], [1, 128, 256, 300, 84], [300, 0, 300], [127, 129, 128]):
        ids = torch.cat([torch.full((c,), v, dtype=torch.int64) for v, c in enumerate(counts)]).to(DEV)
        for order in (ids, ids.flip(0), ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(3)).to(DEV)]):
            gy = made((len(ids), 72), dtype, 4)
            got = ops.embedding_backward(gy, order, len(counts))
            for v, c in enumerate(counts):
                rows = gy[order == v].double()
                tol = (c + 8) * U * rows.abs().sum(0) + HALF_STEP[dtype] * rows.sum(0).abs() + 1e-37
                assert ((got[v].double() - rows.sum(0)).abs() <= tol).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_nothing_to_do(dtype):
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    assert ops.embedding(made((5, 8), dtype, 0), empty).shape == (0, 8)
    assert not ops.embedding_backward(made((0, 9), dtype, 0), empty, 5).any()
    assert ops.embedding_backward(made((3, 8), dtype, 0), torch.zeros(3, dtype=torch.int64, device=DEV), 0).shape == (0, 8)
    nowhere = torch.tensor([-1, 7, 1 << 40], device=DEV)
    assert not ops.embedding(made((5, 8), dtype, 0), nowhere).any()
    assert not ops.embedding_backward(made((3, 8), dtype, 0), nowhere, 5).any()
    assert not ops.embedding(made((0, 8), dtype, 0), nowhere).any()


def test_what_is_not_finite_stays_in_its_row():
    gy = made((600, 16), torch.float32, 5)
    ids = torch.arange(600, device=DEV) % 3
    gy[4, 2], gy[5, 3] = float("nan"), float("inf")
    got = ops.embedding_backward(gy, ids, 4)
    bad = torch.zeros(4, 16, dtype=torch.bool, device=DEV)
    bad[1, 2], bad[2, 3] = True, True
    assert torch.equal(~torch.isfinite(got), bad) and torch.isnan(got[1, 2]) and got[2, 3] == float("inf")
    assert not got[3].any()


def test_shapes_and_autograd():
    table = made((20, 24), torch.float32, 6).requires_grad_()
    ids = torch.tensor([[3, 3, -1], [0, 19, 3]], device=DEV)
    y = ops.embedding(table, ids, scale=2.0)
    assert y.shape == (2, 3, 24)
    gy = made((2, 3, 24), torch.float32, 7)
    got, = torch.autograd.grad(y, table, gy)
    want = torch.zeros(20, 24, device=DEV)
    want[3] = 2 * (gy[0, 0] + gy[0, 1] + gy[1, 2])
    want[0], want[19] = 2 * gy[1, 0], 2 * gy[1, 1]
    assert torch.allclose(got, want, rtol=1e-6, atol=1e-6)
