"""A transformer over a batch of graphs as it is used: embedding rows, blocks of norm, projection, attention, projection
and feed-forward, a readout by attention, and the gradients of all of it."""
import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import layers, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LENGTHS = [23, 1, 40, 64, 9, 0, 31]
HIDDEN, HEADS, KV, DIM, FF, VOCAB = 48, 4, 2, 16, 80, 37


def weights(dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda *s, scale=None: (torch.randn(*s, generator=gen, device=DEV) * (scale or s[0] ** -0.5)).to(dtype)  # noqa: E731
    w = {"table": make(VOCAB, HIDDEN, scale=0.3), "seed": make(len(LENGTHS), HEADS, DIM, scale=1.0)}
    for i in range(2):
        w.update({f"n1{i}": 1 + make(HIDDEN, scale=0.1), f"wqkv{i}": make(HIDDEN, (HEADS + 2 * KV) * DIM), f"bqkv{i}": make((HEADS + 2 * KV) * DIM, scale=0.1),
                  f"wo{i}": make(HEADS * DIM, HIDDEN), f"bo{i}": make(HIDDEN, scale=0.1), f"n2{i}": 1 + make(HIDDEN, scale=0.1),
                  f"wg{i}": make(HIDDEN, FF), f"wu{i}": make(HIDDEN, FF), f"wd{i}": make(FF, HIDDEN)})
    w["wkv"] = make(HIDDEN, 2 * KV * DIM)
    return w


def inputs():
    gen = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(-1, VOCAB, (sum(LENGTHS),), generator=gen, device=DEV)
    bounds = torch.tensor([sum(LENGTHS[:i]) for i in range(len(LENGTHS) + 1)], device=DEV)
    return ids, bounds, torch.arange(len(LENGTHS) + 1, device=DEV)


def net(w, causal):
    ids, p, one_each = inputs()
    h = ops.embedding(w["table"], ids, scale=HIDDEN ** 0.5)
    for i in range(2):
        h = layers.attention_block(h, p, w[f"n1{i}"], (w[f"wqkv{i}"], w[f"bqkv{i}"], w[f"wo{i}"], w[f"bo{i}"]), w[f"n2{i}"],
                                   (w[f"wg{i}"], w[f"wu{i}"], w[f"wd{i}"]), heads=HEADS, kv_heads=KV, causal=causal, activation="gelu")
    kv = ops.linear_act(h, w["wkv"]).view(-1, 2 * KV, DIM)
    return h, ops.segment_attention(w["seed"], kv[:, :KV], kv[:, KV:], one_each, p)


def wide_attention(q, k, v, lengths_q, lengths_k, causal):
    out, a, c = [], 0, 0
    group = q.shape[1] // k.shape[1]
    for n, m in zip(lengths_q, lengths_k):
        kk, vv = (t[c:c + m].repeat_interleave(group, 1) for t in (k, v))
        if m == 0:
            out.append(torch.zeros_like(q[a:a + n]))
        else:
            s = torch.einsum("ihd,jhd->hij", q[a:a + n], kk) * DIM ** -0.5
            if causal:
                s = s.masked_fill(~torch.ones(n, m, dtype=torch.bool, device=DEV).tril(m - n), -float("inf"))
            out.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vv))
        a, c = a + n, c + m
    return torch.cat(out)


def wide_net(w, causal):
    ids, _, _ = inputs()
    rms = lambda x, g: x / (x.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * g     # noqa: E731
    h = torch.where((ids >= 0).unsqueeze(1), w["table"][ids.clamp(min=0)] * HIDDEN ** 0.5, torch.zeros((), dtype=torch.float64, device=DEV))
    for i in range(2):
        x = (rms(h, w[f"n1{i}"]) @ w[f"wqkv{i}"] + w[f"bqkv{i}"]).view(-1, HEADS + 2 * KV, DIM)
        a = wide_attention(x[:, :HEADS], x[:, HEADS:HEADS + KV], x[:, HEADS + KV:], LENGTHS, LENGTHS, causal)
        h = h + a.reshape(-1, HEADS * DIM) @ w[f"wo{i}"] + w[f"bo{i}"]
        y = rms(h, w[f"n2{i}"])
        h = h + (F.gelu(y @ w[f"wg{i}"]) * (y @ w[f"wu{i}"])) @ w[f"wd{i}"]
    kv = (h @ w["wkv"]).view(-1, 2 * KV, DIM)
    return h, wide_attention(w["seed"], kv[:, :KV], kv[:, KV:], [1] * len(LENGTHS), LENGTHS, False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.1)])
def test_a_network_and_its_gradients(dtype, tol, causal):
    """fp32: 2e-5 of the largest value, some 40 roundings of sums of at most 80 terms (2^-24 x 80 x 4 = 2e-5); bf16: each of
    the 16 roundings on the way to a gradient is 2^-8 at most, 0.06 of the largest value, and their products."""
    w = weights(dtype)
    leaves = {n: t.requires_grad_() for n, t in w.items()}
    wide = {n: t.detach().double().requires_grad_() for n, t in w.items()}
    got, want = net(leaves, causal), wide_net(wide, causal)
    for a, b in zip(got, want):
        assert a.shape == b.shape
        assert (a.double() - b).abs().max() <= tol * b.abs().max()
    gen = torch.Generator(device=DEV).manual_seed(8)
    grads = [torch.randn(t.shape, generator=gen, device=DEV) for t in got]
    a = torch.autograd.grad(got, list(leaves.values()), [g.to(dtype) for g in grads])
    b = torch.autograd.grad(want, list(wide.values()), [g.to(dtype).double() for g in grads])
    for n, x, y in zip(leaves, a, b):
        assert (x.double() - y).norm() <= tol * y.norm(), n
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(net(w, causal), got))


def test_recorded():
    w = weights(torch.bfloat16)
    with torch.no_grad():
        net(w, True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        ids, p, one = inputs()
        block = lambda h: layers.attention_block(h, p, w["n10"], (w["wqkv0"], w["bqkv0"], w["wo0"], None), w["n20"],  # noqa: E731
                                                 (w["wg0"], w["wu0"], w["wd0"]), heads=HEADS, kv_heads=KV, causal=True)
        table = w["table"]
        block(ops.embedding(table, ids))
        grad = torch.randn(len(ids), HIDDEN, device=DEV).bfloat16()
        ops.embedding_backward(grad, ids, VOCAB)
        gy = torch.randn(len(ids), HEADS * DIM + 2 * KV * DIM, device=DEV).bfloat16()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            h = ops.embedding(table, ids)
            held = (block(h), ops.embedding_backward(grad, ids, VOCAB), *ops.linear_act_backward(gy, h, w["wqkv0"], w["bqkv0"], "gelu"))
        for i in range(4):
            ids.copy_(torch.randint(-1, VOCAB, ids.shape, device=DEV))
            grad.normal_()
            h = ops.embedding(table, ids)
            want = (block(h), ops.embedding_backward(grad, ids, VOCAB), *ops.linear_act_backward(gy, h, w["wqkv0"], w["bqkv0"], "gelu"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_weights_in_8_bits():
    """The feed-forward half in 8 bits takes the rows of the norm as its own path does."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    make = lambda *s: (torch.randn(*s, generator=gen, device=DEV) * s[0] ** -0.5).bfloat16()   # noqa: E731
    h, p = make(60, 128), torch.tensor([0, 20, 60], device=DEV)
    att, ff = (make(128, 6 * 32), None, make(64, 128), None), [make(128, 256), make(128, 256), make(256, 128)]
    norm = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    got = layers.attention_block(h, p, norm, att, norm, [ops.quantize_weight_fp8(w) for w in ff], heads=2)
    want = layers.attention_block(h, p, norm, att, norm, ff, heads=2)
    assert (got.double() - want.double()).norm() <= 0.1 * want.double().norm()
