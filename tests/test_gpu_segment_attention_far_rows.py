"""Rows of q, k and v that lie more than 16 MB apart, as the first places of long padded sequences do, and a single row with any stride."""
import pytest
import torch

from graphiler_amd import ops
from test_gpu_segment_attention import made, pointer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 20])
@pytest.mark.parametrize("rows", [1, 5])
def test_far_rows(rows, dim, dtype):
    heads, p = 4, pointer([rows])
    apart = (1 << 24) // dtype.itemsize + 8

    def far(t):
        return torch.empty(rows * apart, dtype=dtype, device=DEV).as_strided(t.shape, (apart, dim, 1)).copy_(t)

    q, k, v, grad = (made(rows, heads, dim, dtype, s) for s in range(4))
    out, lse = ops.segment_attention(q, k, v, p, return_lse=True)
    want = ops.segment_attention_backward(grad, q, k, v, out, lse, p)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        a, b, c = (far(t) if w else t for t, w in zip((q, k, v), which))
        assert torch.equal(ops.segment_attention(a, b, c, p), out)
        assert all(torch.equal(x, y) for x, y in zip(ops.segment_attention_backward(grad, a, b, c, out, lse, p), want))
    leaves = [far(t).requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(ops.segment_attention(*leaves, p), leaves, far(grad))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
