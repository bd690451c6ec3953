"""How far bf16 results of attention inside segments, and the gradients of projections, may be off beside their own rounding."""
import math

import pytest
import torch

from graphiler_amd import ops
from segment_attention_bounds import reference
from test_gpu_linear_act import operands
from test_gpu_linear_act import made as made2
from test_gpu_segment_attention import made, pointer

pytestmark = pytest.mark.gpu

# A sum of products with operands that are rounded to bf16 has, where its terms have either sign, the same relative error once more as its
# own rounding to bf16 leaves: each term's error is that of a rounding, independent of the others', and they add up as the terms themselves
# do, by their squares.  Both together sqrt(2) times one rounding.  A tenth is for the chance of a case's values and for the 32-bit sums.
ONCE_MORE = 1.1 * math.sqrt(2)


def off(got, want):
    """In roundings of the result."""
    return float((got.double() - want).norm() / (want.bfloat16().double() - want).norm())


@pytest.mark.parametrize("q_len,k_len,causal,heads,kv_heads", [([900, 500], None, True, 4, 4), ([900, 500], None, False, 8, 2), ([400], [3000], True, 4, 2),
                                                               ([200, 130, 257], None, False, 64, 64), ([60, 40, 33] * 20, None, False, 8, 4)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention(q_len, k_len, causal, heads, kv_heads, dim):
    """Weights are an operand of the result and of grad_v, ds one of grad_q and grad_k; delta adds nothing of bf16's size."""
    keys = k_len or q_len
    q, grad = made(sum(q_len), heads, dim, torch.bfloat16, 5), made(sum(q_len), heads, dim, torch.bfloat16, 8)
    k, v = made(sum(keys), kv_heads, dim, torch.bfloat16, 6), made(sum(keys), kv_heads, dim, torch.bfloat16, 7)
    qp, kp = pointer(q_len), pointer(k_len) if k_len else None
    want = reference(q, k, v, q_len, keys, causal, None, grad)
    out, lse = ops.segment_attention(q, k, v, qp, kp, causal=causal, return_lse=True)
    assert off(out, want[0]) <= ONCE_MORE
    for name, got, w in zip("qkv", ops.segment_attention_backward(grad, q, k, v, out, lse, qp, kp, causal=causal), want[3]):
        assert off(got, w) <= ONCE_MORE, name


@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,m", [(300, 200, 512), (2000, 512, 1024), (5000, 256, 96)])
def test_projection(rows, k, m, act):
    """dz is an operand of all three; without an activation it is grad_y, which has been rounded already."""
    x, w, b, r = operands(rows, k, m, torch.bfloat16, True, True)
    gy = made2((rows, m), torch.bfloat16, 9)
    args = [t.double().requires_grad_() for t in (x, w, b)]
    z = args[0] @ args[1] + args[2]
    y = z if act is None else getattr(torch.nn.functional, act)(z)
    assert off(ops.linear_act(x, w, bias=b, activation=act, residual=r), (y + r.double()).detach()) <= 1.1
    want = torch.autograd.grad(y, args, gy.double())
    for name, got, t in zip(("x", "weight", "bias"), ops.linear_act_backward(gy, x, w, bias=b, activation=act), want):
        assert off(got, t) <= (1.1 if act is None else ONCE_MORE), name
