"""Projections in every form of tile that their sizes can choose, against the definition in 64 bits.  The rules that choose are written
down here again, so that a size which no longer takes the tile it stands for is found."""
import pytest
import torch

from test_gpu_linear_act import check_forward

pytestmark = pytest.mark.gpu


def tiles(rows, cols, high, wide):
    return -(-rows // high) * -(-cols // wide)


def fp32_tile(rows, cols):
    """(parts of 32 rows, wavefronts) of a product that cuts x on the way; None: another kernel's."""
    if rows <= 16 or tiles(rows, cols, 64, 64) <= 512:
        return None
    waves = 4 if (cols - 1) % 256 < 128 else 8
    at_once = 256 if waves == 8 else 512
    cost = {parts: -(-tiles(rows, cols, 32 * parts, 32 * waves) // at_once) * (parts + 1) for parts in range(1, 5 if waves == 8 else 3)}
    return max(p for p in cost if cost[p] == min(cost.values())), waves


@pytest.mark.parametrize("rows,m,tile", [(130, 11111, (1, 4)), (150, 11136, (1, 4)), (131, 10905, (1, 8)), (160, 11264, (1, 8)), (32783, 1, (2, 4)),
                                         (65600, 100, (2, 4)), (10972, 130, (2, 8)), (2000, 2000, (2, 8)), (9000, 512, (3, 8)), (16510, 129, (3, 8)),
                                         (4100, 2047, (3, 8)), (25420, 129, (4, 8)), (16384, 1024, (4, 8))])
def test_fp32_tiles(rows, m, tile):
    assert fp32_tile(rows, m) == tile
    for k in (1, 31, 32, 33, 100, 192):
        check_forward(rows, k, m, torch.float32, "gelu" if k == 33 else None)
    check_forward(rows, 70, m, torch.float32, "silu", bias=False)
    check_forward(rows, 70, m, torch.float32, "relu", residual=False)
