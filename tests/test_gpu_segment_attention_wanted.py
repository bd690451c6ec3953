"""Gradients of attention inside segments that are not wanted are not formed, and the others do not depend on that."""
import itertools

import pytest
import torch

from graphiler_amd import capi, ops
from test_gpu_segment_attention import made, pointer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOTH = [torch.bfloat16, torch.float32]
SOME = [w for w in itertools.product((False, True), repeat=3) if any(w)]
# wavefronts apart, single, sharing tiles; keys of their own; heads that share keys in parts
CASES = [([70, 40], None, 2, 2), ([40, 33, 20, 0, 1] * 3, None, 4, 2), ([200, 130, 257], None, 64, 64), ([3, 1], [500, 90], 8, 1),
         ([300, 200], None, 8, 2)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [20, 32, 64, 128])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", CASES)
def test_each_alone_and_in_pairs(q_len, k_len, heads, kv_heads, dim, causal, dtype):
    keys = k_len or q_len
    qp, kp = pointer(q_len), pointer(k_len) if k_len else None
    tensors = [made(sum(q_len), heads, dim, dtype, 0), made(sum(keys), kv_heads, dim, dtype, 1), made(sum(keys), kv_heads, dim, dtype, 2)]
    grad = made(sum(q_len), heads, dim, dtype, 3)
    out, lse = ops.segment_attention(*tensors, qp, kp, causal=causal, return_lse=True)
    want = ops.segment_attention_backward(grad, *tensors, out, lse, qp, kp, causal=causal)
    for wanted in SOME:
        leaves = [t.clone().requires_grad_(w) for t, w in zip(tensors, wanted)]
        got = torch.autograd.grad(ops.segment_attention(*leaves, qp, kp, causal=causal), [t for t in leaves if t.requires_grad], grad)
        assert all(torch.equal(a, b) for a, b in zip(got, [g for g, w in zip(want, wanted) if w])), wanted


@pytest.mark.parametrize("wanted", SOME)
def test_no_memory_for_what_is_not_wanted(wanted):
    q, k, v = (made(n, 8, 64, torch.bfloat16, s) for s, n in enumerate((40_000, 40_000, 40_000)))
    p = torch.arange(0, 40_001, 100, device=DEV)
    leaves = [t.requires_grad_(w) for t, w in zip((q, k, v), wanted)]
    out = ops.segment_attention(*leaves, p)
    grad = torch.ones_like(out)
    lib = capi.load()
    n = lib.ga_segment_attention_backward_workspace_bytes(400, 40_000, 40_000, 8, 8, 64, capi.GA_BF16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], grad)
    size = out.numel() * 2
    assert torch.cuda.max_memory_allocated() - before < sum(wanted) * size + n + size // 2 and len(got) == sum(wanted)
