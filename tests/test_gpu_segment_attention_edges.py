"""Attention inside segments where it can go wrong: rows in no segment, values that are not finite in masked places, strides,
streams, recorded graphs, gradients through torch, keys far into a long cache."""
import pytest
import torch

from graphiler_amd import ops
from segment_attention_bounds import reference, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOTH = [torch.bfloat16, torch.float32]
NAN, INF = float("nan"), float("inf")


def made(rows, heads, dim, dtype, seed):
    return torch.randn(rows, heads, dim, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def pointer(*bounds):
    return torch.tensor(bounds, dtype=torch.int64, device=DEV)


def both_ways(q, k, v, grad, qp, kp=None, **how):
    out, lse = ops.segment_attention(q, k, v, qp, kp, return_lse=True, **how)
    return (out, lse, *ops.segment_attention_backward(grad, q, k, v, out, lse, qp, kp, **how))


FORMS = [([70, 40], 2), ([40, 33, 20] * 3, 4), ([200, 130, 257], 64)]     # wavefronts apart, single, sharing tiles


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads", FORMS)
def test_rows_in_no_segment(lengths, heads, causal, dtype):
    """NaN in front of the first and behind the last segment reaches nothing; those rows give zeros."""
    first, n = 5, sum(lengths)
    rows = first + n + 9
    q, k, v, grad = (made(rows, heads, 40, dtype, s) for s in range(4))
    bounds = [first]
    for length in lengths:
        bounds.append(bounds[-1] + length)
    inside = slice(first, first + n)
    want = both_ways(*(t[inside].contiguous() for t in (q, k, v, grad)), pointer(*(b - first for b in bounds)), causal=causal)
    for t in (q, k, v, grad):
        t[:first] = NAN
        t[first + n:] = NAN
    got = both_ways(q, k, v, grad, pointer(*bounds), causal=causal)
    for i, (a, b) in enumerate(zip(got, want)):
        if i == 1:
            assert torch.equal(a[:, inside], b)
            assert (a[:, :first] == -INF).all() and (a[:, first + n:] == -INF).all()
        else:
            assert torch.equal(a[inside], b)
            assert not a[:first].any() and not a[first + n:].any()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("lengths,heads", FORMS)
def test_what_is_not_finite_behind_a_query_does_not_reach_it(lengths, heads, bad, dtype):
    """Causal: row j of a value or a key that is not finite leaves the queries in front of j as they were, bit by bit, and
    what sees it is not finite where the definition says so."""
    n = sum(lengths)
    start, length = sum(lengths[:1]), lengths[1]
    j = start + length // 2
    q, k, v, grad = (made(n, heads, 40, dtype, s) for s in range(4))
    bounds = [0]
    for m in lengths:
        bounds.append(bounds[-1] + m)
    p = pointer(*bounds)
    clean = both_ways(q, k, v, grad, p, causal=True)
    hit = v.clone()
    hit[j, :, 3] = bad
    out, lse = ops.segment_attention(q, k, hit, p, causal=True, return_lse=True)
    reached = torch.zeros(n, heads, 40, dtype=torch.bool, device=DEV)
    reached[j:start + length, :, 3] = True
    assert torch.equal(~torch.isfinite(out), reached) and torch.equal(out[~reached], clean[0][~reached])
    assert torch.equal(lse, clean[1])
    if bad == bad:
        assert (out[reached] == bad).all()
    # a key: scores of the queries that see it are not finite; those in front and other segments stay
    hit = k.clone()
    hit[j, :, 3] = bad
    got = both_ways(q, hit, v, grad, p, causal=True)
    apart = torch.ones(n, dtype=torch.bool, device=DEV)
    apart[j:start + length] = False
    for i in (0, 2):
        assert torch.equal(got[i][apart], clean[i][apart])
    apart[start:start + length] = False
    for i in (3, 4):
        assert torch.equal(got[i][apart], clean[i][apart])
    # a gradient row that is not finite: its own query's and its segment's keys up to it, no other
    hit = grad.clone()
    hit[j, :, 3] = bad
    got = ops.segment_attention_backward(hit, q, k, v, *clean[:2], p, causal=True)
    behind = torch.ones(n, dtype=torch.bool, device=DEV)
    behind[start:j + 1] = False
    assert torch.equal(got[1][behind], clean[3][behind]) and torch.equal(got[2][behind], clean[4][behind])
    assert not torch.isfinite(got[2][start:j + 1, :, 3]).any()
    behind[start:j] = True
    assert torch.equal(got[0][behind], clean[2][behind])


@pytest.mark.parametrize("dtype", BOTH)
def test_every_stride(dtype):
    """Columns of one projection, heads in front of rows, a start at an odd value, rows that are all the same."""
    n, h, d = 90, 4, 64
    p = pointer(0, 50, 90)
    fused = made(n, 3 * h, d, dtype, 0)
    q, k, v = fused[:, :h], fused[:, h:2 * h], fused[:, 2 * h:]
    grad = made(n, h, d, dtype, 1)
    want = both_ways(*(t.contiguous() for t in (q, k, v, grad)), p, causal=True)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t)         # noqa: E731
    by_head = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)                                      # noqa: E731
    wide = lambda t: torch.cat([t, t], 2)[:, :, :d]                                                         # noqa: E731
    for form in (lambda t: t, odd, by_head, wide):
        got = both_ways(form(q), form(k), form(v), form(grad), p, causal=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b) and a.is_contiguous()
    one = made(1, h, d, dtype, 2).expand(n, h, d)
    assert torch.equal(ops.segment_attention(q, one, one, p), ops.segment_attention(q, one.contiguous(), one.contiguous(), p))
    narrow = made(n, 3 * h, 21, dtype, 3)                  # rows that are no whole pieces
    parts = [narrow[:, i * h:(i + 1) * h] for i in range(3)]
    for a, b in zip(both_ways(*parts, grad[:, :, :21], p), both_ways(*(t.contiguous() for t in parts), grad[:, :, :21].contiguous(), p)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 32), (4, 1, 20)])
def test_autograd(heads, kv_heads, dim, dtype):
    p = pointer(0, 30, 75)
    q, k, v = (made(75, h, dim, dtype, i).requires_grad_() for i, h in enumerate((heads, kv_heads, kv_heads)))
    grad = made(75, heads, dim, dtype, 5)
    out, lse = ops.segment_attention(q, k, v, p, causal=True, return_lse=True)
    got = torch.autograd.grad(out, (q, k, v), grad)
    want = ops.segment_attention_backward(grad, q.detach(), k.detach(), v.detach(), out.detach(), lse, p, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    fused = made(75, heads + 2 * kv_heads, dim, dtype, 6).requires_grad_()
    out = ops.segment_attention(fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:], p)
    assert torch.autograd.grad(out.float().sum(), fused)[0].shape == fused.shape
    if dtype == torch.float32:                             # against differences of the definition in 64 bits
        for i, g in enumerate(got):
            args = [t.detach().double() for t in (q, k, v)]
            step = torch.randn_like(args[i])
            at = []
            for sign in (1, -1):
                moved = [a + sign * 1e-5 * step if j == i else a for j, a in enumerate(args)]
                at.append((_wide(*moved, [30, 45]) * grad.double()).sum())
            slope = (at[0] - at[1]) / 2e-5
            assert abs(slope - (g.double() * step).sum()) <= 1e-4 * (g.double() * step).abs().sum()


def _wide(q, k, v, lengths):
    out, a = torch.zeros_like(q), 0
    group = q.shape[1] // k.shape[1]
    for n in lengths:
        seen = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        for h in range(q.shape[1]):
            s = q[a:a + n, h] @ k[a:a + n, h // group].t() * q.shape[2] ** -0.5
            out[a:a + n, h] = torch.softmax(s.masked_fill(~seen, -INF), 1) @ v[a:a + n, h // group]
        a += n
    return out


@pytest.mark.parametrize("dtype", BOTH)
def test_recorded_and_replayed(dtype):
    """Both directions in a graph, with keys cut into parts, rows laid out and shared heads in parts; every replay
    with other inputs, against the eager result, with eager work between."""
    cases = [((3, 2, 64, [1, 1, 2], [3000, 900, 2100], False), 6), ((0, 4, 20, [90, 60], [90, 60], True), 8),
             ((1, 2, 128, [40] * 5, [40] * 5, True), 2)]
    for (seed, kv, dim, q_len, k_len, causal), heads in cases:
        qp = pointer(*[sum(q_len[:i]) for i in range(len(q_len) + 1)])
        kp = pointer(*[sum(k_len[:i]) for i in range(len(k_len) + 1)])
        q, grad = made(sum(q_len), heads, dim, dtype, seed), made(sum(q_len), heads, dim, dtype, seed + 1)
        k, v = made(sum(k_len), kv, dim, dtype, seed + 2), made(sum(k_len), kv, dim, dtype, seed + 3)
        both_ways(q, k, v, grad, qp, kp, causal=causal)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both_ways(q, k, v, grad, qp, kp, causal=causal)
        for i in range(4):
            for j, t in enumerate((q, k, v, grad)):
                t.copy_(made(*t.shape, dtype, 100 * i + j))
            want = both_ways(q, k, v, grad, qp, kp, causal=causal)
            for t in held:
                t.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_gradients_are_not_recorded():
    q = made(20, 2, 16, torch.float32, 0).requires_grad_()
    p = pointer(0, 20)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        with torch.cuda.graph(graph):
            ops.segment_attention(q, q, q, p)
    torch.cuda.synchronize()


def test_another_stream():
    p = pointer(0, 300, 500)
    q, k, v, grad = (made(500, 4, 64, torch.bfloat16, s) for s in range(4))
    want = both_ways(q, k, v, grad, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both_ways(q, k, v, grad, p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", BOTH)
def test_keys_far_into_a_long_cache(dtype):
    """Keys behind 4 GiB of others, and values there; bounds behind the rows are the last row."""
    h, d = 4, 128
    rows = (5 << 30) // (h * d * (2 if dtype == torch.bfloat16 else 4))
    k, v = (torch.zeros(rows, h, d, dtype=dtype, device=DEV) for _ in range(2))
    k[-1000:], v[-1000:] = made(1000, h, d, dtype, 0), made(1000, h, d, dtype, 1)
    q = made(3, h, d, dtype, 2)
    got = ops.segment_attention(q, k, v, pointer(0, 1, 3), pointer(rows - 1000, rows - 400, rows + 5))
    want = ops.segment_attention(q, k[-1000:].contiguous(), v[-1000:].contiguous(), pointer(0, 1, 3), pointer(0, 600, 1000))
    want64 = reference(q, k[-1000:], v[-1000:], [1, 2], [600, 400], False)
    within(got, want64[0], want64[1])
    within(want, want64[0], want64[1])


def test_refusals():
    q, p = made(10, 4, 16, torch.float32, 0), pointer(0, 10)
    k2, wide = made(10, 3, 16, torch.float32, 0), made(10, 4, 136, torch.float32, 0)
    for call, what in ((lambda: ops.segment_attention(q, k2, k2, p), "divisor"), (lambda: ops.segment_attention(q, q[:5], q[:5], p), "q's rows"),
                       (lambda: ops.segment_attention(wide, wide, wide, p), "at most 128"),
                       (lambda: ops.segment_attention(q, q.bfloat16(), q, p), "dtype"), (lambda: ops.segment_attention(q.half(), q.half(), q.half(), p), "float32 or bfloat16"),
                       (lambda: ops.segment_attention(q, q, q, p.int()), "int64"), (lambda: ops.segment_attention(q, q, q, p.cpu()), "CUDA"),
                       (lambda: ops.segment_attention(q, q, q, p, pointer(0, 5, 10)), "one entry more"),
                       (lambda: ops.segment_attention(q, q, q, p, scale=0.0), "scale"), (lambda: ops.segment_attention(q, q, q, p, scale=NAN), "scale"),
                       (lambda: ops.segment_attention(q[:, :, ::2], q[:, :, ::2], q[:, :, ::2], p), "contiguous"),
                       (lambda: ops.segment_attention_backward(q, q, q, q, q, torch.zeros(10, 4, device=DEV), p), "lse"),
                       (lambda: ops.segment_attention_backward(q[:5], q, q, q, q, torch.zeros(4, 10, device=DEV), p), "grad_out")):
        with pytest.raises(RuntimeError, match=what):
            call()
    assert ops.segment_attention(q[:0], q[:0], q[:0], pointer(0)).shape == (0, 4, 16)
    assert not ops.segment_attention(q, q[:0], q[:0], p, pointer(0, 0)).any()
