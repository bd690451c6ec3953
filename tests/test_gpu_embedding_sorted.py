"""The embedding gradient of more places than one launch looks through: sorted, summed in runs of 64 places and joined.  Every width of
lanes, rows that begin and end at the cuts, values that are not finite, recorded graphs."""
import pytest
import torch

from graphiler_amd import capi, ops
from test_gpu_embedding import BOTH, DEV, HALF_STEP, U, check, made

pytestmark = pytest.mark.gpu
RUN = 64


def sorted_path(n, rows, cols):
    """Few places need no workspace; the sort does."""
    return capi.load().ga_embedding_backward_workspace_bytes(n, rows, cols) > 0


def sums_of(gy, ids, rows):
    """(sums, sums of magnitudes, counts) in 64 bits."""
    there = ((ids >= 0) & (ids < rows)).unsqueeze(1)
    safe = ids.long().clamp(0, rows - 1)
    g = gy.double() * there
    sums = torch.zeros(rows, gy.shape[1], dtype=torch.float64, device=DEV)
    mags, counts = torch.zeros_like(sums), torch.zeros(rows, 1, dtype=torch.float64, device=DEV)
    sums.index_add_(0, safe, g)
    mags.index_add_(0, safe, g.abs())
    counts.index_add_(0, safe, there.double())
    return sums, mags, counts


def near(got, gy, ids, rows, dtype):
    sums, mags, counts = sums_of(gy, ids, rows)
    tol = (counts + 8) * U * mags + HALF_STEP[dtype] * sums.abs() * (1 + 1e-6) + 1e-37
    off = (got.double() - sums).abs()
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("cols", [1, 7, 8, 15, 63, 64, 65, 72, 100, 127, 128, 129, 200, 256, 257, 300, 513, 1500])
def test_widths(cols, dtype):
    for n, rows in ((1100, 9), (3000, 90), (1025, 70000)):
        assert sorted_path(n, rows, cols)
        check(n, rows, cols, dtype)
        check(n, rows, cols, dtype, bits=32, skew=4.0, scale=-0.3)


COUNTS = [[63] * 20, [64] * 20, [65] * 20, [127, 1] * 10, [128] * 10, [129, 63] * 8, [1, 64, 65, 62] * 8, [0, 130, 0, 62, 0, 128] * 6,
          [32, 64, 64, 64, 32] * 5, [1, 2000], [2000, 1], [64, 1300, 64], [1, 63, 1300, 61, 3], [5000]]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("cols", [7, 64, 100, 200, 513])
def test_rows_that_begin_and_end_at_the_cuts_and_next_to_them(cols, dtype):
    """Rows of the table that 63, 64, 65, 127, 128 and 129 places name, from a cut on and from others: in order, backwards, mixed
    and behind 1, 37 or 64 places that name no row."""
    for counts in COUNTS:
        ids = torch.cat([torch.full((c,), v, dtype=torch.int64) for v, c in enumerate(counts)])
        mixed = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(3))]
        for order in (ids, ids.flip(0), mixed, torch.cat([torch.full((37,), -1), ids, torch.full((64,), len(counts))])):
            order = order.to(DEV)
            assert sorted_path(len(order), len(counts), cols)
            gy = made((len(order), cols), dtype, 4)
            got = ops.embedding_backward(gy, order, len(counts))
            near(got, gy, order, len(counts), dtype)
            assert torch.equal(got, ops.embedding_backward(gy, order, len(counts)))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("cols", [16, 65, 129, 300])
def test_what_is_not_finite_stays_in_its_row(cols, dtype):
    """In rows of few places, of many and next to each other in a run; behind ids outside the table nothing is read."""
    counts = [3, 500, 1, 64, 700, 40]
    ids = torch.cat([torch.full((c,), v, dtype=torch.int64) for v, c in enumerate(counts)] + [torch.tensor([-1, 6])])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(8))].to(DEV)
    assert sorted_path(len(ids), 6, cols)
    gy = made((len(ids), cols), dtype, 5)
    gy[(ids < 0) | (ids >= 6)] = float("nan")
    want = ops.embedding_backward(gy, ids, 6)
    assert torch.isfinite(want).all()
    for row, col, bad in ((0, 2, float("nan")), (1, 3, float("inf")), (4, cols - 1, -float("inf")), (5, 0, float("nan"))):
        gy[torch.nonzero(ids == row)[-1, 0], col] = bad
    gy[torch.nonzero(ids == 1)[0, 0], 4], gy[torch.nonzero(ids == 1)[-1, 0], 4] = float("inf"), -float("inf")
    got = ops.embedding_backward(gy, ids, 6)
    bad = torch.zeros(6, cols, dtype=torch.bool, device=DEV)
    bad[0, 2] = bad[1, 3] = bad[1, 4] = bad[4, cols - 1] = bad[5, 0] = True
    assert torch.equal(~torch.isfinite(got), bad) and torch.equal(got[~bad], want[~bad])
    assert torch.isnan(got[0, 2]) and got[1, 3] == float("inf") and torch.isnan(got[1, 4])
    assert got[4, cols - 1] == -float("inf") and torch.isnan(got[5, 0])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,rows,cols", [(1500, 40, 72), (5000, 300, 65), (20000, 7, 200), (3000, 70000, 24), (40000, 3000, 513)])
def test_recorded_and_replayed(n, rows, cols, dtype):
    """Every replay with other ids and rows, against the eager result, with eager work between."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    ids = torch.randint(-1, rows + 1, (n,), generator=gen, device=DEV)
    gy = made((n, cols), dtype, 0)
    assert sorted_path(n, rows, cols)
    ops.embedding_backward(gy, ids, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.embedding_backward(gy, ids, rows)
    for i in range(4):
        gy.copy_(made((n, cols), dtype, 10 + i))
        spread = torch.rand(n, generator=gen, device=DEV).pow(1 + i) * (rows + 2) - 1
        ids.copy_(spread.long().clamp(-1, rows))
        want = ops.embedding_backward(gy, ids, rows)
        held.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        near(held, gy, ids, rows, dtype)


@pytest.mark.parametrize("dtype", BOTH)
def test_rows_at_any_address(dtype):
    """grad_y that begins at an odd value: rows of every alignment."""
    for n, rows, cols in ((1300, 11, 65), (1300, 11, 64), (1300, 800, 129)):
        gen = torch.Generator(device=DEV).manual_seed(cols)
        ids = torch.randint(0, rows, (n,), generator=gen, device=DEV)
        gy = made((n, cols), dtype, 6)
        odd = torch.empty(n * cols + 1, dtype=dtype, device=DEV)[1:].view(n, cols).copy_(gy)
        assert torch.equal(ops.embedding_backward(gy, ids, rows), ops.embedding_backward(odd, ids, rows))


def test_a_scale_that_is_not_finite_is_refused():
    table, ids = made((5, 8), torch.float32, 0), torch.tensor([0, -1], device=DEV)
    for scale in (float("inf"), float("nan")):
        for call in (lambda: ops.embedding(table, ids, scale=scale), lambda: ops.embedding_backward(table[:2], ids, 5, scale=scale)):
            with pytest.raises(RuntimeError, match="scale must be finite"):
                call()
