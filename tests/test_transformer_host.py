"""Refusals of attention inside segments, of projections and of embedding rows, without a GPU: the C entry points
return before they launch, the Python operators raise before they call."""
import pytest
import torch
from torch.autograd import forward_ad

from graphiler_amd import capi, layers, ops

PTR = 1 << 20            # a pointer that is aligned and never followed
EINVAL, EUNSUPPORTED, EWORKSPACE, EALIGN = -1, -2, -3, -4
BF16, F32 = capi.GA_BF16, capi.GA_F32


def attention(q=PTR, q_row=512, q_head=64, k=PTR, k_row=256, k_head=64, v=PTR, v_row=256, v_head=64, qp=PTR, kp=PTR, segments=3,
              out=PTR, lse=PTR, nq=10, nk=20, heads=8, kv_heads=4, dim=64, causal=0, scale=0.1, dt=BF16, ws=PTR, size=None):
    lib = capi.load()
    if size is None:
        size = lib.ga_segment_attention_workspace_bytes(segments, nq, nk, heads, kv_heads, dim, dt)
    return lib.ga_segment_attention(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, qp, kp, segments, out, lse, nq, nk,
                                    heads, kv_heads, dim, causal, scale, dt, ws, size, None)


def backward(go=PTR, q=PTR, q_row=512, k=PTR, v=PTR, out=PTR, lse=PTR, qp=PTR, kp=PTR, segments=3, gq=PTR, gk=PTR, gv=PTR, nq=10,
             nk=20, heads=8, kv_heads=4, dim=64, scale=0.1, dt=BF16, ws=PTR, size=None):
    lib = capi.load()
    if size is None:
        size = lib.ga_segment_attention_backward_workspace_bytes(segments, nq, nk, heads, kv_heads, dim, dt)
    return lib.ga_segment_attention_backward(go, q, q_row, 64, k, 256, 64, v, 256, 64, out, lse, qp, kp, segments, gq, gk, gv, nq, nk,
                                             heads, kv_heads, dim, 0, scale, dt, ws, size, None)


def test_attention_codes():
    assert attention(nq=0) == 0
    for bad in (dict(nq=-1), dict(nk=-1), dict(segments=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0),
                dict(q=None), dict(k=None), dict(v=None), dict(qp=None), dict(kp=None), dict(out=None), dict(scale=0.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(q_row=-8)):
        assert attention(**bad) == EINVAL, bad
    for bad in (dict(dt=7), dict(dim=129), dict(dim=136), dict(heads=1 << 17, kv_heads=1), dict(nk=1 << 31), dict(nq=1 << 30),
                dict(q_row=1 << 26), dict(k_row=1 << 26), dict(segments=1 << 31)):
        assert attention(**bad, size=1 << 40) == EUNSUPPORTED, bad
    for bad in (dict(k=PTR + 2), dict(v=PTR + 8), dict(k_row=260), dict(v_head=68), dict(out=PTR + 1), dict(lse=PTR + 2),
                dict(qp=PTR + 4), dict(q=PTR + 1), dict(q=PTR + 2, dt=F32)):
        assert attention(**bad) == EALIGN, bad


def test_attention_workspaces():
    lib = capi.load()
    small = lib.ga_segment_attention_workspace_bytes
    assert small(3, 10, 20, 8, 4, 64, BF16) == 0
    laid = small(3, 10, 20, 8, 4, 60, BF16)               # rows that are not whole pieces are laid out
    assert laid == 2 * 20 * 4 * 128                       # 60 values take 8 pieces
    assert attention(dim=60, ws=None) == EWORKSPACE and attention(dim=60, size=laid - 1) == EWORKSPACE
    assert attention(dim=60, ws=PTR + 8) == EWORKSPACE
    parts = small(16, 16, 16 * 8192, 32, 4, 128, BF16)    # one query a segment: its keys are cut
    assert parts > 0 and parts % (16 * 32 * 130 * 4) == 0
    assert small(3, 10, 20, 8, 3, 64, BF16) == 0 and small(3, 10, 20, 8, 4, 300, BF16) == 0
    n = lib.ga_segment_attention_backward_workspace_bytes(3, 10, 20, 8, 4, 64, BF16)
    assert n >= 10 * 8 * 4


def test_attention_backward_codes():
    for bad in (dict(go=None), dict(out=None), dict(lse=None), dict(gq=None), dict(gk=None), dict(gv=None), dict(nq=-1),
                dict(scale=0.0), dict(kv_heads=5), dict(qp=None)):
        assert backward(**bad) == EINVAL, bad
    assert backward(dim=200) == EUNSUPPORTED and backward(dt=4) == EUNSUPPORTED
    for bad in (dict(go=PTR + 2), dict(q=PTR + 2), dict(k=PTR + 4), dict(q_row=516), dict(gq=PTR + 1), dict(lse=PTR + 1)):
        assert backward(**bad) == EALIGN, bad
    assert backward(ws=None) == EWORKSPACE and backward(size=8) == EWORKSPACE and backward(ws=PTR + 4) == EWORKSPACE


@pytest.mark.parametrize("dt", [F32, BF16])
def test_linear_act_codes(dt):
    lib = capi.load()
    rows, k, m = 20_000, 65, 333
    n = lib.ga_linear_act_workspace_bytes(rows, k, m, dt)
    assert n > 0 and lib.ga_linear_act_workspace_bytes(3, k, m, dt) == 0
    assert lib.ga_linear_act_workspace_bytes(rows, 64, 64, BF16) == 0

    def call(x=PTR, w=PTR, b=PTR, r=PTR, y=PTR, rows=rows, k=k, m=m, act=0, dt=dt, ws=PTR, size=n):
        return lib.ga_linear_act(x, w, b, r, y, rows, k, m, act, dt, ws, size, None)

    assert call(rows=0) == 0
    for bad in (dict(rows=-1), dict(k=0), dict(m=0), dict(x=None), dict(w=None), dict(y=None)):
        assert call(**bad) == EINVAL, bad
    assert call(act=9) == EUNSUPPORTED and call(act=-2) == EUNSUPPORTED and call(dt=4) == EUNSUPPORTED
    assert call(k=(1 << 20) + 1) == EUNSUPPORTED and call(m=(1 << 20) + 1) == EUNSUPPORTED
    assert call(ws=None) == EWORKSPACE and call(size=n - 1) == EWORKSPACE and call(ws=PTR + 8) == EWORKSPACE
    for bad in (dict(x=PTR + 1), dict(b=PTR + 1), dict(r=PTR + 1), dict(y=PTR + 1)):
        assert call(**bad) == EALIGN, bad
    if dt == BF16:
        assert call(x=PTR + 2, k=64, m=64) == EALIGN
    assert call(rows=1 << 40, k=64, m=64, size=1 << 50) == EUNSUPPORTED
    size = lib.ga_linear_act_backward_workspace_bytes(rows, k, m, 0, dt)
    assert size > 0 and lib.ga_linear_act_backward_workspace_bytes(rows, k, m, 7, dt) == 0

    def back(gy=PTR, x=PTR, w=PTR, b=None, gx=PTR, gw=PTR, gb=None, rows=rows, act=0, dt=dt, ws=PTR, size=size):
        return lib.ga_linear_act_backward(gy, x, w, b, gx, gw, gb, rows, k, m, act, dt, ws, size, None)

    assert back(gy=None) == EINVAL and back(x=None) == EINVAL and back(w=None) == EINVAL and back(rows=-3) == EINVAL
    assert back(act=5) == EUNSUPPORTED and back(gx=PTR + 1) == EALIGN and back(gb=PTR + 1) == EALIGN
    assert back(ws=None) == EWORKSPACE and back(size=size - 1) == EWORKSPACE


def test_embedding_codes():
    lib = capi.load()

    def call(t=PTR, ids=PTR, bits=64, y=PTR, n=5, rows=10, cols=8, dt=BF16):
        return lib.ga_embedding(t, ids, bits, y, n, rows, cols, 1.0, dt, None)

    assert call(n=0) == 0
    for bad in (dict(n=-1), dict(rows=-1), dict(cols=0), dict(bits=16), dict(ids=None), dict(y=None), dict(t=None)):
        assert call(**bad) == EINVAL, bad
    assert call(dt=9) == EUNSUPPORTED and call(cols=(1 << 20) + 1) == EUNSUPPORTED and call(n=1 << 42) == EUNSUPPORTED
    assert call(t=PTR + 1) == EALIGN and call(ids=PTR + 4) == EALIGN and call(ids=PTR + 2, bits=32) == EALIGN
    size = lib.ga_embedding_backward_workspace_bytes(5000, 10, 8)
    assert lib.ga_embedding_backward_workspace_bytes(5, 10, 8) == 0        # few places need none
    assert size > 0 and lib.ga_embedding_backward_workspace_bytes(1 << 31, 10, 8) == 0

    def back(gy=PTR, ids=PTR, bits=64, g=PTR, n=5, rows=10, cols=8, dt=BF16, ws=PTR, size=size):
        return lib.ga_embedding_backward(gy, ids, bits, g, n, rows, cols, 1.0, dt, ws, size, None)

    assert back(rows=0) == 0
    assert back(gy=None) == EINVAL and back(g=None) == EINVAL and back(ids=None) == EINVAL and back(bits=8) == EINVAL
    assert back(n=1 << 31) == EUNSUPPORTED and back(rows=1 << 31) == EUNSUPPORTED
    assert back(n=5000, ws=None) == EWORKSPACE and back(n=5000, ws=PTR + 64) == EWORKSPACE
    assert back(n=5000, size=size - 1) == EWORKSPACE


def test_operators_refuse_host_tensors_and_names():
    q, p, x, w = torch.randn(6, 2, 8), torch.tensor([0, 6]), torch.randn(3, 8), torch.randn(8, 4)
    ids = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.segment_attention(q, q, q, p), lambda: ops.segment_attention_backward(q, q, q, q, q, q, p),
                 lambda: ops.linear_act(x, w), lambda: ops.linear_act_backward(x, x, w), lambda: ops.embedding(x, ids),
                 lambda: ops.embedding_backward(x, ids, 4),
                 lambda: layers.attention_block(x, p, x[0], (torch.randn(8, 24), None, w, None), x[0], (w, w, w), heads=2)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="activation"):
        ops.linear_act(x, w, activation="tanh")
    with pytest.raises(RuntimeError, match="heads a multiple of kv_heads"):
        layers.attention_block(x, p, x[0], (torch.randn(8, 24), None, w, None), x[0], (w, w, w), heads=3, kv_heads=2)
    with pytest.raises(RuntimeError, match="column for each value"):
        layers.attention_block(x, p, x[0], (torch.randn(8, 25), None, w, None), x[0], (w, w, w), heads=2)
    with pytest.raises(RuntimeError, match="8 bits"):
        layers.attention_block(x, p, x[0], (torch.randn(8, 24), None, w, None), x[0], (w, (w, w), w), heads=2)


def test_tangents_and_traces_are_refused():
    x, w = torch.randn(3, 8), torch.randn(8, 4)
    q, p, ids = torch.randn(6, 2, 8), torch.tensor([0, 6]), torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual, dual3 = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: ops.linear_act(dual, w), lambda: ops.embedding(dual, ids),
                     lambda: ops.segment_attention(dual3, q, q, p)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda a: ops.linear_act(a, w), (x,))
