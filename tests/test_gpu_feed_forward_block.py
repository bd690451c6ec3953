"""An HGT layer with its norms, residual stream and feed-forward block, as the operators are used together,
against the same composition in float64 around the attention layer; refusals of what the operators cannot take."""
import pytest
import torch
import torch.nn.functional as F

from graphiler_amd import datasets, layers, ops, prepare_graph
from graphiler_amd.hipgraph import Graphed

pytestmark = pytest.mark.gpu


def network(device, dtype, hidden, heads, ff, seed=0):
    wl = datasets.hgt_hetero(counts=(400, 300, 200, 101), edges_per_type=1500)
    g = prepare_graph(wl.src, wl.dst, wl.num_nodes, device=device, ntype_of=wl.ntype, num_ntypes=4,
                      etype_of=wl.etype, num_etypes=10)
    gen = torch.Generator().manual_seed(seed)
    nt, ne, d = 4, 10, hidden // heads

    def draw(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=gen)).to(dtype).to(device)

    h = draw(wl.num_nodes, hidden)
    attention = [draw(nt, hidden, hidden, scale=hidden ** -0.5) for _ in range(4)]
    attention += [draw(ne, heads, d, d, scale=d ** -0.5) for _ in range(2)]
    attention += [torch.rand(ne, heads, generator=gen).to(device), torch.randn(nt, generator=gen).to(device)]
    norms = [(1 + 0.2 * torch.randn(hidden, generator=gen)).to(dtype).to(device) for _ in range(2)]
    weights = (draw(hidden, ff, scale=hidden ** -0.5), draw(hidden, ff, scale=hidden ** -0.5),
               draw(ff, hidden, scale=ff ** -0.5))
    return g, h, norms, attention, weights


def norm64(t, w):
    return t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6) * w.double()


def block64(h, a, norms, weights):
    t = h.double() + a.double()
    x = norm64(t, norms[1])
    wg, wu, wd = (w.double() for w in weights)
    return t + (F.silu(x @ wg) * (x @ wu)) @ wd


@pytest.mark.parametrize("dtype,hidden,heads,ff", [(torch.float32, 64, 2, 170), (torch.bfloat16, 128, 4, 344),
                                                   (torch.bfloat16, 128, 2, 341)])
def test_block_against_float64(device, dtype, hidden, heads, ff):
    g, h, norms, attention, weights = network(device, dtype, hidden, heads, ff)
    out = layers.hgt_block(g, h, norms[0], attention, norms[1], weights, heads=heads)
    assert out.shape == h.shape and out.dtype == dtype
    a = layers.hgt_layer(g, ops.rms_norm(h, norms[0]), *attention, heads=heads)
    want = block64(h, a, norms, weights)
    off = ((out.double() - want).norm() / want.norm()).item()
    # roundings side by side: norm, hidden rows, down projection, residual; fp32: sums of random signs
    assert off <= (4 * torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 2.0 ** -19), off


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_in_8_bits(device, dtype):
    g, h, norms, attention, weights = network(device, dtype, 128, 4, 300)
    weights8 = tuple(ops.quantize_weight_fp8(w) for w in weights)
    out = layers.hgt_block(g, h, norms[0], attention, norms[1], weights8, heads=4)
    a = layers.hgt_layer(g, ops.rms_norm(h, norms[0]), *attention, heads=4)
    want = block64(h, a, norms, weights)
    t = h.double() + a.double()
    # the feed-forward half goes through rows and weights of 2^-4 steps twice; the stream does not
    assert ((out.double() - want).norm() / (want - t).norm()).item() <= 4 * 2.0 ** -4
    # and it is the operators one after the other
    x8, s, total = ops.rms_norm_fp8(a, norms[1], residual=h)
    hidden = ops.gated_linear_fp8(x8, s, *weights8[0], *weights8[1], out_dtype=dtype)
    same = total + ops.linear_fp8(*ops.quantize_fp8(hidden), *weights8[2], out_dtype=dtype)
    assert torch.equal(out, same)
    rows = ops.rms_norm(a, norms[1], residual=h)[0]
    assert layers.feed_forward(rows, *weights8).dtype == dtype


def test_block_replays_in_a_graph(device):
    g, h, norms, attention, weights = network(device, torch.bfloat16, 128, 4, 344)
    weights8 = tuple(ops.quantize_weight_fp8(w) for w in weights)

    def step():
        mid = layers.hgt_block(g, h, norms[0], attention, norms[1], weights, heads=4)
        return layers.hgt_block(g, mid, norms[0], attention, norms[1], weights8, heads=4)

    recorded = Graphed(step)
    for seed in range(4):
        h.copy_(torch.randn(h.shape, generator=torch.Generator().manual_seed(seed)))
        got = recorded().clone()
        assert torch.equal(got, step())


def test_training_step_of_a_feed_forward_half(device):
    """Gradients of norm, residual and gated block together, against float64's."""
    gen = torch.Generator().manual_seed(3)
    h, a = (torch.randn(300, 96, generator=gen).to(device) for _ in range(2))
    w = (1 + 0.1 * torch.randn(96, generator=gen)).to(device)
    wg, wu = (torch.randn(96, 200, generator=gen).to(device) / 10 for _ in range(2))
    wd = torch.randn(200, 96, generator=gen).to(device) / 14
    leaves = [t.requires_grad_() for t in (h, a, w, wg, wu, wd)]
    x, t = ops.rms_norm(a, w, residual=h)
    (t + torch.mm(ops.gated_linear(x, wg, wu), wd)).pow(2).sum().backward()
    wide = [t.detach().double().requires_grad_() for t in leaves]
    t64 = wide[0] + wide[1]
    x64 = t64 / torch.sqrt((t64 * t64).mean(1, keepdim=True) + 1e-6) * wide[2]
    (t64 + (F.silu(x64 @ wide[3]) * (x64 @ wide[4])) @ wide[5]).pow(2).sum().backward()
    for got, want in zip(leaves, wide):
        assert ((got.grad.double() - want.grad).norm() / want.grad.norm()).item() <= 2.0 ** -18


def test_gradients_are_the_same_with_two_streams_and_no_order(device):
    x = torch.randn(2000, 72, device=device).bfloat16()
    w = [torch.randn(72, 96, device=device).bfloat16() for _ in range(2)]
    gh = torch.randn(2000, 96, device=device).bfloat16()
    first = ops.gated_linear_backward(gh, x, *w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.gated_linear_backward(gh, x, *w))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for other in got:
        for p, q in zip(first, other):
            assert torch.equal(p, q)


@pytest.mark.parametrize("rows,m", [(300, 32), (20000, 48), (50, 130)])
def test_gradients_of_a_feed_forward_block(device, rows, m):
    """Those of the last weight too, at sizes whose product without gradients is the framework's own kernel."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 96, generator=gen).to(device)
    wg, wu = (torch.randn(96, 200, generator=gen).to(device) / 10 for _ in range(2))
    wd = torch.randn(200, m, generator=gen).to(device) / 14
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    out = layers.feed_forward(*leaves)
    out.pow(2).sum().backward()
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ((F.silu(wide[0] @ wide[1]) * (wide[0] @ wide[2])) @ wide[3]).pow(2).sum().backward()
    for got, want in zip(leaves, wide):
        assert ((got.grad.double() - want.grad).norm() / want.grad.norm()).item() <= 2.0 ** -18
    with torch.no_grad():
        again = layers.feed_forward(*leaves)
    assert ((again - out).norm() / out.norm()).item() <= 2.0 ** -18


def test_refusals(device):
    x, w = torch.randn(4, 64, device=device), torch.ones(64, device=device)
    wide = torch.randn(64, 32, device=device)
    x8, s = ops.quantize_fp8(x)
    w8, ws = ops.quantize_weight_fp8(wide)
    refused = [
        lambda: ops.rms_norm(x.t(), w), lambda: ops.rms_norm(x, w[:63]), lambda: ops.rms_norm(x, w.bfloat16()),
        lambda: ops.rms_norm(x, w, x[:3]), lambda: ops.rms_norm(x.half(), w.half()), lambda: ops.rms_norm(x[0], w),
        lambda: ops.rms_norm(x, w, eps=-1.0), lambda: ops.rms_norm(x, w, eps=float("nan")),
        lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(x[:, :0], w[:0]),
        lambda: ops.rms_norm(torch.zeros(1, 16385, device=device), torch.ones(16385, device=device)),
        lambda: ops.rms_norm_fp8(x.clone().requires_grad_(), w), lambda: ops.quantize_fp8(x[:, ::2]),
        lambda: ops.rms_norm_backward(x[:3], x, w), lambda: ops.rms_norm_backward(x, x, w, grad_sum=x.bfloat16()),
        lambda: ops.quantize_weight_fp8(wide.clone().requires_grad_()), lambda: ops.quantize_weight_fp8(w),
        lambda: ops.linear_fp8(x, s, w8, ws), lambda: ops.linear_fp8(x8, s[:3], w8, ws),
        lambda: ops.linear_fp8(x8, s, w8, ws.cpu()), lambda: ops.linear_fp8(x8, s, w8[:, :64].contiguous(), ws),
        lambda: ops.linear_fp8(x8, s, w8, ws, out_dtype=torch.float16),
        lambda: ops.linear_fp8(x8, s.view(torch.uint8), w8, ws),
        lambda: ops.gated_linear_fp8(x8, s, w8, ws, w8[:31].contiguous(), ws),
        lambda: ops.gated_linear(x, wide, wide[:, :31].contiguous()), lambda: ops.gated_linear(x, wide.t(), wide.t()),
        lambda: ops.gated_linear(x, wide.bfloat16(), wide.bfloat16()), lambda: ops.gated_linear(x, wide, wide, "tanh"),
        lambda: ops.gated_linear_backward(x, x, wide, wide), lambda: ops.gated_linear(x, wide, wide.cpu()),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(f"call {i} was taken")
