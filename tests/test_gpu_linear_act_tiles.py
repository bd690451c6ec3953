"""Projections in every form of tile that their sizes can choose, against the definition in 64 bits.  The rules that choose are written
down here again, so that a size which no longer takes the tile it stands for is found."""
import pytest
import torch

from test_gpu_linear_act import check_backward, check_forward

pytestmark = pytest.mark.gpu


def tiles(rows, cols, high, wide):
    return -(-rows // high) * -(-cols // wide)


def bf16_tile(rows, cols):
    """Rows (and columns) of a tile of one bf16 product."""
    large, small = tiles(rows, cols, 256, 256), tiles(rows, cols, 128, 128)
    if small <= 512:
        return 64 if small <= 256 else 128
    return 256 if 115 * large * (-(-small // 512) * 512) >= 100 * small * (-(-large // 256) * 256) else 128


def fp32_tile(rows, cols):
    """(parts of 32 rows, wavefronts) of a product that cuts x on the way; None: another kernel's."""
    if rows <= 16 or tiles(rows, cols, 64, 64) <= 512:
        return None
    waves = 4 if (cols - 1) % 256 < 128 else 8
    at_once = 256 if waves == 8 else 512
    cost = {parts: -(-tiles(rows, cols, 32 * parts, 32 * waves) // at_once) * (parts + 1) for parts in range(1, 5 if waves == 8 else 3)}
    return max(p for p in cost if cost[p] == min(cost.values())), waves


# the last 256 columns whole, more than 128 of them (whole eights, odd, whole fours) and fewer (whole eights, odd, whole fours)
@pytest.mark.parametrize("m", [4096, 4040, 4001, 3972, 3912, 3913, 3844])
@pytest.mark.parametrize("k", [72, 200])
def test_bf16_tiles_of_256_columns_as_two_of_128(m, k):
    rows = 8192
    assert bf16_tile(rows, m) == bf16_tile(rows, -(-m // 8) * 8) == 256
    check_forward(rows, k, m, torch.bfloat16, "gelu")
    check_forward(rows, k, m, torch.bfloat16, None, bias=False)
    check_forward(rows, k, m, torch.bfloat16, None, residual=False)
    check_backward(rows, k, m, torch.bfloat16, "silu")
    check_backward(rows, k, m, torch.bfloat16, "relu", bias=False)


def test_bf16_tiles_of_256_columns_at_a_row_that_ends_inside():
    rows, k, m = 8191, 70, 4001
    assert bf16_tile(rows, m) == bf16_tile(rows, 4008) == 256
    check_forward(rows, k, m, torch.bfloat16, "relu")
    check_backward(rows, k, m, torch.bfloat16, "gelu")


@pytest.mark.parametrize("rows,m,tile", [(130, 11111, (1, 4)), (150, 11136, (1, 4)), (131, 10905, (1, 8)), (160, 11264, (1, 8)), (32783, 1, (2, 4)),
                                         (65600, 100, (2, 4)), (10972, 130, (2, 8)), (2000, 2000, (2, 8)), (9000, 512, (3, 8)), (16510, 129, (3, 8)),
                                         (4100, 2047, (3, 8)), (25420, 129, (4, 8)), (16384, 1024, (4, 8))])
def test_fp32_tiles(rows, m, tile):
    assert fp32_tile(rows, m) == tile
    for k in (1, 31, 32, 33, 100, 192):
        check_forward(rows, k, m, torch.float32, "gelu" if k == 33 else None)
    check_forward(rows, 70, m, torch.float32, "silu", bias=False)
    check_forward(rows, 70, m, torch.float32, "relu", residual=False)
