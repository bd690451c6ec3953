"""Attention inside segments in 64 bits, and how far a kernel of 32-bit sums may be from it.

Bounds of one output, from the sizes alone (u = 2^-24, half a step of fp32; r half a step of the tensors' type):
  a score of D products and its factors is off by (D + 4) u of the sum of the products' magnitudes; the
  logarithm of a sum of n exponentials adds (n + 8) u; so a weight p is off by
      e = 2 (D + 4) u S + 2 (|s| + 8) u + (n + 8) u  of itself   (S: the largest such sum, |s| <= S),
  plus r where it is rounded as an operand (bf16).  A sum of n weighed values is off by (n + 8) u of the sum of its
  terms' magnitudes besides, and its result by r of itself.
"""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def visible(n, m, causal, device):
    seen = torch.ones(n, m, dtype=torch.bool, device=device)
    return seen.tril(m - n) if causal else seen


def reference(q, k, v, q_len, k_len, causal, scale=None, grad=None, q_first=0, k_first=0):
    """(out, its bound, lse[, three gradients, their bounds]) in float64, a segment and head at a time."""
    dtype, dev = q.dtype, q.device
    r = HALF_STEP[dtype]
    operand = r if dtype == torch.bfloat16 else 0.0
    groups, d = q.shape[1] // k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    out, out_tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((q.shape[1], q.shape[0]), -float("inf"), dtype=torch.float64, device=dev)
    grads = tols = None
    if grad is not None:
        g = grad.detach().double()
        grads = [torch.zeros_like(t) for t in (q, k, v)]
        tols = [torch.zeros_like(t) for t in (q, k, v)]
        summed = [torch.zeros_like(t) for t in (q, k, v)]          # magnitudes of the terms
    a, c = q_first, k_first
    for n, m in zip(q_len, k_len):
        seen = visible(n, m, causal, dev)
        some = seen.any(dim=1) if m else torch.zeros(n, dtype=torch.bool, device=dev)
        for h in range(q.shape[1]):
            if n == 0 or m == 0:
                continue
            x, y, z = q[a:a + n, h], k[c:c + m, h // groups], v[c:c + m, h // groups]
            s = (x @ y.t()) * scale
            s = torch.where(seen, s, torch.full_like(s, -float("inf")))
            top = s.amax(dim=1, keepdim=True)
            p = torch.exp(s - torch.where(some.unsqueeze(1), top, torch.zeros_like(top)))
            total = p.sum(dim=1, keepdim=True)
            p = torch.where(some.unsqueeze(1), p / total, torch.zeros_like(p))
            lse[h, a:a + n] = torch.where(some, top[:, 0] + total[:, 0].log(), lse[h, a:a + n])
            size = ((x.abs() @ y.abs().t()) * abs(scale)).where(seen, torch.zeros_like(s)).amax(dim=1, keepdim=True)
            e = 2 * (d + 4) * U * size + 2 * (size + 8) * U + (m + 8) * U
            o, mag = p @ z, p @ z.abs()
            out[a:a + n, h] = o
            out_tol[a:a + n, h] = (e + operand + (m + 8) * U) * mag + r * o.abs() + 1e-37
            if grad is None:
                continue
            gi = g[a:a + n, h]
            dp, delta = gi @ z.t(), (gi * o).sum(dim=1, keepdim=True)
            ds = p * (dp - delta)
            if dtype == torch.bfloat16:          # delta is the sum of the weighed dp, whose products are off as the scores' are
                delta_off = ((e + (m + 8) * U) * p * dp.abs() + (d + 8) * U * p * (gi.abs() @ z.abs().t())).sum(dim=1, keepdim=True)
            else:                                # ... of the products with out
                delta_off = (gi.abs() * out_tol[a:a + n, h]).sum(dim=1, keepdim=True)
            off = p * (e * (dp.abs() + delta.abs()) + (d + 8) * U * (gi.abs() @ z.abs().t()) + (d + 8) * U * (gi.abs() * o.abs()).sum(1, keepdim=True)
                       + delta_off) + 4 * U * ds.abs()
            off = off + operand * (ds.abs() + off)
            terms = abs(scale) * (ds.abs() @ y.abs())
            grads[0][a:a + n, h] += scale * (ds @ y)
            tols[0][a:a + n, h] += abs(scale) * (off @ y.abs())
            summed[0][a:a + n, h] += terms
            grads[1][c:c + m, h // groups] += scale * (ds.t() @ x)
            tols[1][c:c + m, h // groups] += abs(scale) * (off.t() @ x.abs())
            summed[1][c:c + m, h // groups] += abs(scale) * (ds.abs().t() @ x.abs())
            grads[2][c:c + m, h // groups] += p.t() @ gi
            tols[2][c:c + m, h // groups] += ((e + operand) * p).t() @ gi.abs()
            summed[2][c:c + m, h // groups] += p.t() @ gi.abs()
        a, c = a + n, c + m
    if grad is None:
        return out, out_tol, lse
    longest = max([1, *q_len, *k_len]) * groups
    tols = [t + (longest + 8) * U * s + r * x.abs() + 1e-37 for t, s, x in zip(tols, summed, grads)]
    return out, out_tol, lse, grads, tols


def within(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound, worst {float((off / tol)[bad].max()):.3g} times it"
