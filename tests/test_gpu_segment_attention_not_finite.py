"""Attention inside segments with keys and queries that are not finite: what reaches the gradients is the same in tiles that an
edge cuts and in whole ones."""
import pytest
import torch

from graphiler_amd import ops
from segment_attention_bounds import reference, within
from test_gpu_segment_attention import made, pointer

pytestmark = pytest.mark.gpu
BOTH = [torch.bfloat16, torch.float32]
INF = float("inf")
# wavefronts apart, single, sharing tiles: tiles that an edge cuts, and whole ones
FORMS = [([70, 40], 2), ([128, 64], 2), ([40, 33, 20] * 3, 4), ([64] * 4, 4), ([200, 130, 257], 64), ([256, 128, 384], 64)]


def both_ways(q, k, v, grad, p, k_pointer=None, causal=False):
    out, lse = ops.segment_attention(q, k, v, p, k_pointer, causal=causal, return_lse=True)
    return (out, lse, *ops.segment_attention_backward(grad, q, k, v, out, lse, p, k_pointer, causal=causal))


def inputs(lengths, heads, dim, dtype):
    n = sum(lengths)
    q, k, v, grad = (made(n, heads, dim, dtype, s) for s in range(4))
    return q, k, v, grad


def without(t, j):
    return torch.cat([t[:j], t[j + 1:]])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [32, 40, 128])
@pytest.mark.parametrize("lengths,heads", FORMS)
@pytest.mark.parametrize("last", [False, True])
def test_a_key_whose_scores_are_minus_infinity(last, lengths, heads, dim, dtype):
    """Its weight is 0 and grad_q's terms of it are 0 k: NaN in the columns where k is infinite, 0 in the others."""
    q, k, v, grad = inputs(lengths, heads, dim, dtype)
    q[:, :, 3] = q[:, :, 3].abs() + 0.5
    j, s = sum(lengths[:1]) + (lengths[1] - 1 if last else lengths[1] // 2), 1
    k[j, :, 3] = -INF
    out, lse, gq, gk, gv = both_ways(q, k, v, grad, pointer(lengths))
    less = [n - (i == s) for i, n in enumerate(lengths)]
    want, tol, want_lse, grads, tols = reference(q, without(k, j), without(v, j), lengths, less, False, None, grad)
    within(out, want, tol, "out")
    assert ((lse.double() - want_lse).abs() <= 1e-4 + 2e-5 * want_lse.abs()).all()
    within(without(gk, j), grads[1], tols[1], "gradient of k")
    within(without(gv, j), grads[2], tols[2], "gradient of v")
    assert not gk[j].any() and not gv[j].any()
    seen = torch.zeros_like(gq, dtype=torch.bool)
    seen[sum(lengths[:s]):sum(lengths[:s + 1]), :, 3] = True
    assert torch.equal(torch.isnan(gq), seen)
    within(gq.masked_fill(seen, 0), grads[0].masked_fill(seen, 0), tols[0], "gradient of q")


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [32, 40, 128])
@pytest.mark.parametrize("lengths,heads", FORMS)
@pytest.mark.parametrize("last", [False, True])
def test_a_query_whose_scores_are_minus_infinity(last, lengths, heads, dim, dtype):
    """It has weights of 0, zeros as its result and a log-sum-exp of -inf; grad_k's terms of it are 0 q."""
    q, k, v, grad = inputs(lengths, heads, dim, dtype)
    k[:, :, 3] = k[:, :, 3].abs() + 0.5
    i, s = sum(lengths[:1]) + (lengths[1] - 1 if last else lengths[1] // 2), 1
    q[i, :, 3] = -INF
    out, lse, gq, gk, gv = both_ways(q, k, v, grad, pointer(lengths))
    assert not out[i].any() and (lse[:, i] == -INF).all() and not gq[i].any()
    less = [n - (a == s) for a, n in enumerate(lengths)]
    want, tol, _, grads, tols = reference(without(q, i), k, v, less, lengths, False, None, without(grad, i))
    within(without(out, i), want, tol, "out")
    within(without(gq, i), grads[0], tols[0], "gradient of q")
    within(gv, grads[2], tols[2], "gradient of v")
    seen = torch.zeros_like(gk, dtype=torch.bool)
    seen[sum(lengths[:s]):sum(lengths[:s + 1]), :, 3] = True
    assert torch.equal(torch.isnan(gk), seen)
    within(gk.masked_fill(seen, 0), grads[1].masked_fill(seen, 0), tols[1], "gradient of k")


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [40, 128])
@pytest.mark.parametrize("lengths,heads", FORMS)
def test_only_what_sees_it(lengths, heads, dim, dtype):
    """Causal: the queries in front of such a key, and the keys behind such a query, keep finite gradients."""
    q, k, v, grad = inputs(lengths, heads, dim, dtype)
    p, start, n = pointer(lengths), sum(lengths[:1]), lengths[1]
    j = start + n // 2
    hit, up = k.clone(), q.clone()
    up[:, :, 3] = up[:, :, 3].abs() + 0.5
    hit[j, :, 3] = -INF
    gq = both_ways(up, hit, v, grad, p, causal=True)[2]
    seen = torch.zeros_like(gq, dtype=torch.bool)
    seen[j:start + n, :, 3] = True
    assert torch.equal(torch.isnan(gq), seen)
    hit, up = q.clone(), k.clone()
    up[:, :, 3] = up[:, :, 3].abs() + 0.5
    hit[j, :, 3] = -INF
    gk = both_ways(hit, up, v, grad, p, causal=True)[3]
    seen = torch.zeros_like(gk, dtype=torch.bool)
    seen[start:j + 1, :, 3] = True
    assert torch.equal(torch.isnan(gk), seen)
