"""Attention inside segments against the definition in 64 bits, with bounds that come from the sizes."""
import pytest
import torch

from graphiler_amd import ops
from segment_attention_bounds import reference, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOTH = [torch.bfloat16, torch.float32]


def pointer(lengths, first=0):
    p = [first]
    for n in lengths:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int64, device=DEV)


def made(rows, heads, dim, dtype, seed, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=gen, device=DEV) * scale).to(dtype)


def check(q_len, k_len, heads, kv_heads, dim, causal, dtype, backward=True, scale=None, seed=0, spare=0):
    same = k_len is None
    keys = q_len if same else k_len
    nq, nk = sum(q_len) + spare, sum(keys) + spare
    q, k, v = made(nq, heads, dim, dtype, seed, 1.5), made(nk, kv_heads, dim, dtype, seed + 1), made(nk, kv_heads, dim, dtype, seed + 2)
    grad = made(nq, heads, dim, dtype, seed + 3) if backward else None
    want = reference(q, k, v, q_len, keys, causal, scale, grad)
    qp, kp = pointer(q_len), None if same else pointer(keys)
    out, lse = ops.segment_attention(q, k, v, qp, kp, causal=causal, scale=scale, return_lse=True)
    within(out, want[0], want[1], "out")
    finite = torch.isfinite(want[2])
    assert torch.equal(finite, torch.isfinite(lse)) and (lse[~finite] == -float("inf")).all()
    assert ((lse.double() - want[2])[finite].abs() <= 1e-4 + 2e-5 * want[2][finite].abs()).all()
    assert torch.equal(out, ops.segment_attention(q, k, v, qp, kp, causal=causal, scale=scale))
    if backward:
        got = ops.segment_attention_backward(grad, q, k, v, out, lse, qp, kp, causal=causal, scale=scale)
        for name, g, w, t in zip("qkv", got, want[3], want[4]):
            within(g, w, t, "gradient of " + name)
        again = ops.segment_attention_backward(grad, q, k, v, out, lse, qp, kp, causal=causal, scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


LENGTHS = [[1], [0, 1, 2], [31, 32, 33], [63, 0, 64, 65, 1], [127, 128, 129], [300], [5] * 70, []]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda n: "x".join(map(str, n[:5])) or "none")
def test_lengths(lengths, causal, dtype):
    check(lengths, None, 2, 2, 32, causal, dtype, spare=3)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [1, 3, 8, 16, 20, 33, 40, 64, 72, 96, 100, 128])
def test_widths(dim, dtype):
    check([70, 9, 140], None, 2, 1, dim, False, dtype)
    check([70, 9, 140], None, 1, 1, dim, True, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (4, 2), (6, 2), (8, 1), (16, 4)])
def test_shared_heads(heads, kv_heads, causal, dtype):
    check([40, 130, 3], None, heads, kv_heads, 64, causal, dtype)
    check([1, 1, 1], [200, 77, 0], heads, kv_heads, 64, causal, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len", [([1], [1000]), ([3, 2, 0, 4], [500, 0, 90, 2]), ([200], [30]), ([33, 65], [64, 1]),
                                         ([1] * 5, [4000, 1, 64, 65, 2000]), ([257], [1500])])
def test_queries_and_keys_of_their_own(q_len, k_len, causal, dtype):
    check(q_len, k_len, 4, 2, 64, causal, dtype)
    check(q_len, k_len, 2, 2, 128, causal, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale", [1.0, 0.01, -0.3])
def test_scales(scale, dtype):
    check([100, 29], None, 2, 2, 48, False, dtype, scale=scale)


@pytest.mark.parametrize("dtype", BOTH)
def test_long(dtype):
    check([2500, 1000], None, 2, 1, 128, True, dtype)
    check([1700], None, 1, 1, 64, False, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [24, 64, 128])
def test_enough_workgroups_for_tiles_that_wavefronts_share(dim, causal, dtype):
    """128 rows a workgroup and 256 workgroups at least, on both sides; single wavefronts where segments are short."""
    check([200, 130, 70, 257], None, 64, 64, dim, causal, dtype)
    check([100, 130, 70, 64], [300, 90, 129, 10], 128, 64, dim, causal, dtype, backward=dim < 128)
    check([40, 64, 65, 3, 0, 33, 32] * 10, None, 4, 2, dim, causal, dtype)


@pytest.mark.parametrize("q_len,k_len,causal", [([182, 61, 40, 7], None, True), ([116, 20], None, False), ([3, 2, 3], [179, 64, 20], False),
                                                ([300, 500], None, True)])
@pytest.mark.parametrize("dim", [16, 32])
def test_grad_q_of_narrow_heads_is_off_by_its_own_rounding(q_len, k_len, causal, dim):
    # With few keys that count, a delta from the rounded result or ds of 8 bits would add to it: here delta is a sum in 32 bits and ds
    # has 16, 2^-8 of what the result's rounding is off by.  A tenth is for the 32-bit sums and the weights' exponentials.
    keys = k_len or q_len
    q, k, v = made(sum(q_len), 4, dim, torch.bfloat16, 5, 1.8), made(sum(keys), 2, dim, torch.bfloat16, 6), made(sum(keys), 2, dim, torch.bfloat16, 7)
    grad = made(sum(q_len), 4, dim, torch.bfloat16, 8)
    qp, kp = pointer(q_len), pointer(k_len) if k_len else None
    want = reference(q, k, v, q_len, keys, causal, None, grad)[3][0]
    out, lse = ops.segment_attention(q, k, v, qp, kp, causal=causal, return_lse=True)
    got = ops.segment_attention_backward(grad, q, k, v, out, lse, qp, kp, causal=causal)[0]
    assert (got.double() - want).norm() <= 1.1 * (want.bfloat16().double() - want).norm()
