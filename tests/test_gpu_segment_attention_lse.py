"""Gradients of the log-sum-exps of attention inside segments: d lse_i / d s_ij is the weight p_ij."""
import pytest
import torch

from graphiler_amd import ops
from segment_attention_bounds import HALF_STEP, U, reference, visible, within
from test_gpu_segment_attention import made, pointer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOTH = [torch.bfloat16, torch.float32]
CASES = [([70, 40], None, 2, 2), ([40, 33, 20, 0, 1] * 3, None, 4, 2), ([200, 130, 257], None, 64, 64), ([3, 1, 2], [500, 90, 0], 8, 1),
         ([300, 200], None, 8, 2), ([50], [20], 2, 1)]


def added(q, k, q_len, k_len, causal, glse):
    """What the gradients of the log-sum-exps add to those of q and k, and its bound: with e, the error of a weight (the score's and the
    exponential's, as segment_attention_bounds has it), ds = p glse is off by (e + 4 u) of itself and in bf16 by half a step as an
    operand, and so is each term of a sum."""
    r = HALF_STEP[q.dtype] if q.dtype == torch.bfloat16 else 0.0
    groups, d, scale = q.shape[1] // k.shape[1], q.shape[2], q.shape[2] ** -0.5
    q, k, glse = q.detach().double(), k.detach().double(), glse.detach().double()
    grads, tols = [torch.zeros_like(q), torch.zeros_like(k)], [torch.zeros_like(q), torch.zeros_like(k)]
    a = c = 0
    for n, m in zip(q_len, k_len):
        for h in range(q.shape[1]):
            if n == 0 or m == 0:
                continue
            x, y = q[a:a + n, h], k[c:c + m, h // groups]
            seen = visible(n, m, causal, DEV)
            s = (x @ y.t() * scale).masked_fill(~seen, -float("inf"))
            p = torch.softmax(s, 1).masked_fill(~seen, 0)         # NaN where nothing is seen
            size = (x.abs() @ y.abs().t() * scale).amax(dim=1, keepdim=True)
            e = 2 * (d + 4) * U * size + 2 * (size + 8) * U + (m + 8) * U
            ds = p * glse[h, a:a + n].unsqueeze(1)
            off = ds.abs() * (e + 4 * U + r)
            grads[0][a:a + n, h] += scale * (ds @ y)
            tols[0][a:a + n, h] += scale * (off @ y.abs() + (m + 8) * U * (ds.abs() @ y.abs()))
            grads[1][c:c + m, h // groups] += scale * (ds.t() @ x)
            tols[1][c:c + m, h // groups] += scale * (off.t() @ x.abs() + (n * groups + 8) * U * (ds.abs().t() @ x.abs()))
        a, c = a + n, c + m
    return grads, tols


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [20, 32, 64, 128])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", CASES)
def test_through_autograd(q_len, k_len, heads, kv_heads, dim, causal, dtype):
    keys = k_len or q_len
    qp, kp = pointer(q_len), pointer(k_len) if k_len else None
    q, k, v = (made(sum(n), h, dim, dtype, s).requires_grad_() for s, (n, h) in enumerate(((q_len, heads), (keys, kv_heads), (keys, kv_heads))))
    grad = made(sum(q_len), heads, dim, dtype, 3)
    glse = torch.randn(heads, sum(q_len), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    out, lse = ops.segment_attention(q, k, v, qp, kp, causal=causal, return_lse=True)
    want = reference(q, k, v, q_len, keys, causal, None, grad)
    more, more_tol = added(q, k, q_len, keys, causal, glse)
    r = HALF_STEP[dtype]
    got = torch.autograd.grad((out, lse), (q, k, v), (grad, glse), retain_graph=True)
    for i, name in enumerate("qk"):
        both = want[3][i] + more[i]
        within(got[i], both, want[4][i] + more_tol[i] + r * more[i].abs() + 1e-37, "gradient of " + name)
    within(got[2], want[3][2], want[4][2], "gradient of v")
    # alone
    alone = torch.autograd.grad(lse, (q, k, v), glse)
    for i, name in enumerate("qk"):
        within(alone[i], more[i], more_tol[i] * (1 + 2 * r) + r * more[i].abs() + 1e-37, "gradient of lse to " + name)
    assert not alone[2].any()
    again = ops.segment_attention_backward(grad, q.detach(), k.detach(), v.detach(), out.detach(), lse.detach(), qp, kp, causal=causal, grad_lse=glse)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


def test_against_differences():
    """Of the definition in 64 bits, the loss a function of both results; a gradient that is one value for all."""
    q_len, p = [30, 45], pointer([30, 45])
    q, k, v = (made(75, h, 24, torch.float32, s).requires_grad_() for s, h in enumerate((4, 2, 2)))
    out, lse = ops.segment_attention(q, k, v, p, causal=True, return_lse=True)
    grad = made(75, 4, 24, torch.float32, 5)
    got = torch.autograd.grad((out * grad).sum() + 3 * lse.sum(), (q, k, v))

    def loss(*args):
        o, _, s = reference(args[0].float(), args[1].float(), args[2].float(), q_len, q_len, True)[:3]
        return (o * grad.double()).sum() + 3 * s.sum()

    for i, g in enumerate(got):
        args = [t.detach() for t in (q, k, v)]
        step = torch.randint(-1, 2, args[i].shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV) * 2.0 ** -9
        up, down = ([a + s * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        # both points are rounded to fp32 (2^-24 of values below 8, against steps of 2^-9: 2^-12), the cubes of the steps are left out
        slope, along = loss(*up) - loss(*down), 2 * (g.double() * step)
        assert abs(slope - along.sum()) <= 1e-3 * along.abs().sum()


def test_refusals():
    q, p = made(10, 4, 16, torch.float32, 0), pointer([10])
    out, lse = ops.segment_attention(q, q, q, p, return_lse=True)
    for bad, what in ((lse.t().contiguous(), "heads, queries"), (lse.double(), "float32"), (lse.cpu(), "CUDA"), (lse[:, :5], "heads, queries")):
        with pytest.raises(RuntimeError, match=what):
            ops.segment_attention_backward(out, q, q, q, out, lse, p, grad_lse=bad)


@pytest.mark.parametrize("dtype", BOTH)
def test_recorded_and_replayed(dtype):
    p = pointer([90, 60])
    q, k, v, grad = (made(150, h, 64, dtype, s) for s, h in enumerate((8, 2, 2, 8)))
    glse = torch.randn(8, 150, device=DEV)

    def both():
        out, lse = ops.segment_attention(q, k, v, p, causal=True, return_lse=True)
        return ops.segment_attention_backward(grad, q, k, v, out, lse, p, causal=True, grad_lse=glse)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for i in range(4):
        for j, t in enumerate((q, k, v, grad)):
            t.copy_(made(*t.shape, dtype, 100 * i + j))
        glse.normal_()
        want = both()
        for t in held:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
