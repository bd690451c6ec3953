"""Few queries a segment over many keys, in as many segments as fill the chip: keys cut between wavefronts and, where that leaves
compute units idle, between workgroups."""
import pytest
import torch

from graphiler_amd import capi
from test_gpu_segment_attention import check

BOTH = [torch.bfloat16, torch.float32]


def test_keys_are_cut_for_as_many_segments_as_there_are_compute_units():
    small = capi.load().ga_segment_attention_workspace_bytes
    for dt in (capi.GA_BF16, capi.GA_F32):
        assert small(64, 64, 64 * 8192, 32, 4, 128, dt) == 2 * 64 * 32 * 130 * 4           # two parts: sums, a maximum and a sum each
        assert small(256, 256, 256 * 4096, 32, 4, 128, dt) == 0                            # one, by four wavefronts
        assert small(256, 256, 256 * 512, 32, 4, 128, dt) == 0
        assert small(2048, 2048, 2048 * 8192, 32, 4, 128, dt) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,dim", [(1, 128), (1, 20), (4, 64), (3, 32)])
def test_many_segments_of_few_queries(queries, dim, causal, dtype):
    """1024 or 545 keys a segment on average, some with none, one or few."""
    keys = [1500, 0, 1, 3000, 33, 1100, 64, 2500] * 8
    check([queries] * 64, keys, 32, 4, dim, causal, dtype, backward=False)
    check([queries, 0, 1, queries] * 64, [1024, 7, 50, 1100] * 64, 8, 1, dim, causal, dtype, backward=False)
