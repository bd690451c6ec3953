"""How large embedding rows and their gradient may be, without a GPU: what a launch does not hold is refused before the first one, and
what it holds is not.  So is a scale that would make NaN of the zeros of ids outside the table."""
import pytest
import torch

from graphiler_amd import capi, ops

PTR = 1 << 20            # a pointer that is aligned and never followed
EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3
LANES = [(1, 8), (64, 8), (65, 16), (128, 16), (129, 32), (256, 32), (257, 64), (4096, 64)]


@pytest.mark.parametrize("cols,lanes", LANES)
@pytest.mark.parametrize("dt", [capi.GA_F32, capi.GA_BF16])
def test_the_gradient(cols, lanes, dt):
    lib = capi.load()

    def call(n_ids, n_table):
        return lib.ga_embedding_backward(PTR, PTR, 64, PTR, n_ids, n_table, cols, 1.0, dt, PTR, 0, None)

    blocks = 0xffffffff // 256
    most_ids, most_rows = blocks * 64, blocks * (256 // lanes)
    assert most_ids == (1 << 30) - 64 and most_rows == (1 << 32) // lanes - 256 // lanes
    # held: it goes on to look at the workspace
    assert call(most_ids, 10) == EWORKSPACE and call(5000, most_rows) == EWORKSPACE and call(most_ids, most_rows) == EWORKSPACE
    assert lib.ga_embedding_backward_workspace_bytes(most_ids, most_rows, cols) > 8 * most_ids + 4 * most_rows
    for n_ids, n_table in ((most_ids + 1, 10), ((1 << 31) - 3, 10), (5000, most_rows + 1), (0, most_rows + 1), (1 << 40, 1 << 40)):
        assert call(n_ids, n_table) == EUNSUPPORTED
        assert lib.ga_embedding_backward_workspace_bytes(n_ids, n_table, cols) == 0


@pytest.mark.parametrize("cols,lanes", LANES)
def test_the_lookup(cols, lanes):
    lib = capi.load()
    most = 0xffffffff // 256 * (256 // lanes * 4)
    assert most == (1 << 34) // lanes - 1024 // lanes
    assert lib.ga_embedding(PTR, PTR, 64, PTR, most + 1, 10, cols, 1.0, capi.GA_BF16, None) == EUNSUPPORTED


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan")])
def test_a_scale_that_is_not_finite(scale):
    lib = capi.load()
    assert lib.ga_embedding(PTR, PTR, 64, PTR, 1 << 40, 10, 8, scale, capi.GA_F32, None) == EINVAL
    assert lib.ga_embedding_backward(PTR, PTR, 64, PTR, 5000, 10, 8, scale, capi.GA_F32, PTR, 0, None) == EINVAL
    with pytest.raises(RuntimeError, match="scale must be finite"):
        ops._finite(scale)
    assert ops._finite(torch.tensor(2.0)) == 2.0
