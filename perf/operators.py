"""The operators around an attention layer, as cases that can be timed: the norm of the residual
stream, the matrix product of 8-bit rows, and the gated feed-forward block with its gradients.

A case is one call as a user's program makes it (with ``own``: the framework's operators; without: the
same definition in elementary torch operations, in 32 bits, rounded once at the end).  Rows are
nodes of a graph, or the one to few rows of a query that is answered by itself; the widths are those of
the benchmark's networks and generic powers of two, and odd ones between them.

8-bit values are e4m3; every block of 128 values of a row (of 128 x 128 values of a weight) has a
scale that is a power of two, the smallest one that brings the block's largest magnitude to at
most 448.  A row is padded with zeros to whole blocks.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "bf16": 2}
BLOCK = 128
EPS = 1e-6


def listed():
    return [
        # One node is answered by itself: its row after an attention layer, added to the residual
        # stream and normalised.  The latency of a call is what counts.
        {"name": "norm_one_row", "kind": "norm", "form": "plain", "rows": 1, "cols": 1_024,
         "dtype": "bf16", "residual": True},
        # Every node of the benchmark's social graph between the attention of a layer and its
        # feed-forward block, four heads of 64.
        {"name": "norm_all_nodes", "kind": "norm", "form": "plain", "rows": 232_965, "cols": 256,
         "dtype": "bf16", "residual": True},
        # A wide stream that goes on into 8-bit products: values, scales and the new residual.
        {"name": "norm_8bit_wide", "kind": "norm", "form": "fp8", "rows": 16_384, "cols": 4_096,
         "dtype": "bf16", "residual": True},
        # Training: the gradients of the norm of a citation graph's 500 input features, fp32,
        # with what comes down the residual stream.
        {"name": "norm_gradients", "kind": "norm", "form": "grad", "rows": 19_717, "cols": 500,
         "dtype": "fp32", "residual": True},
        # One row of features is cut to 8 bits and multiplied: all weights are read for it.
        {"name": "fp8_one_row", "kind": "fp8", "form": "linear", "rows": 1, "k": 4_096, "m": 4_096},
        # The gate and the up projection of a citation graph's nodes in 8 bits, an odd number of
        # rows and a width that no tile divides; the rows come out of the norm in 8 bits.
        {"name": "fp8_gated_nodes", "kind": "fp8", "form": "gated", "rows": 19_717, "k": 256,
         "m": 1_000},
        # A large batch of wide rows: the matrix instructions are the bound.
        {"name": "fp8_large", "kind": "fp8", "form": "linear", "rows": 16_384, "k": 4_096, "m": 4_096},
        # Three nodes are answered together through a bf16 feed-forward block.
        {"name": "gated_three_rows", "kind": "gated", "form": "forward", "rows": 3, "k": 1_024,
         "m": 4_096, "dtype": "bf16", "act": "silu"},
        # The smallest citation graph in fp32, hidden width 128, two thirds of four times that.
        {"name": "gated_cora_fp32", "kind": "gated", "form": "forward", "rows": 2_708, "k": 128,
         "m": 341, "dtype": "fp32", "act": "gelu"},
        # A batch of nodes through a wide block.
        {"name": "gated_large", "kind": "gated", "form": "forward", "rows": 16_384, "k": 1_024,
         "m": 4_096, "dtype": "bf16", "act": "silu"},
        # Training of that block: gradients of the rows and of both weights.
        {"name": "gated_train", "kind": "gated", "form": "grad", "rows": 8_192, "k": 1_024,
         "m": 4_096, "dtype": "bf16", "act": "silu"},
        # Training of a small block in fp32, no size a multiple of a tile.
        {"name": "gated_train_fp32", "kind": "gated", "form": "grad", "rows": 2_001, "k": 300,
         "m": 700, "dtype": "fp32", "act": "gelu"},
    ]


# most of what a pass of a drawn case may compute or move
MOST_VALUES = 16_384 * 4_096
MOST_FLOPS = {"fp8": 5.4e11, "bf16": 4.0e11, "fp32": 4.0e10}


def _spread(rng, low, high, step=1):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step))


def _width(rng, low, high):
    """Half of the widths are multiples of 64, the others any number."""
    return _spread(rng, max(low, 64), high, 64) if rng.random() < 0.5 else _spread(rng, low, high)


def draw(rng):
    while True:
        kind = rng.choice(["norm", "fp8", "gated"])
        if kind == "norm":
            case = {"kind": kind, "form": rng.choice(["plain", "plain", "fp8", "grad"]),
                    "rows": _spread(rng, 1, 262_144), "cols": _width(rng, 16, 8_192),
                    "dtype": rng.choice(["bf16", "fp32"]), "residual": rng.random() < 0.7}
            if case["rows"] * case["cols"] * BYTES[case["dtype"]] <= 2 * MOST_VALUES:
                return case
        elif kind == "fp8":
            case = {"kind": kind, "form": rng.choice(["linear", "gated"]), "rows": _spread(rng, 1, 32_768),
                    "k": _width(rng, 64, 8_192), "m": _width(rng, 32, 8_192)}
            if work(case)["flops"] <= MOST_FLOPS["fp8"]:
                return case
        else:
            case = {"kind": kind, "form": rng.choice(["forward", "grad"]), "rows": _spread(rng, 1, 65_536),
                    "k": _width(rng, 32, 2_048), "m": _width(rng, 32, 8_192),
                    "dtype": rng.choice(["bf16", "bf16", "fp32"]),
                    "act": rng.choice(["silu", "gelu", "relu"])}
            if work(case)["flops"] <= MOST_FLOPS[case["dtype"]]:
                return case


# ---- inputs --------------------------------------------------------------------------------------

def _rows(gen, rows, cols, dtype, spread=0.5, scale=1.0):
    """Normal values whose columns differ in size, as the features of a trained network do."""
    width = torch.exp(spread * torch.randn(cols, generator=gen, device=DEV))
    x = torch.randn(rows, cols, generator=gen, device=DEV).mul_(width).mul_(scale)
    return x.to(dtype)


def _weight(gen, k, m, dtype):
    return (torch.randn(k, m, generator=gen, device=DEV) / math.sqrt(k)).to(dtype)


def _weight_8bit(gen, k, m):
    """A weight as the 8-bit product holds it: (m, k padded) values and (m / 128, k / 128) scales."""
    w = _weight(gen, k, m, torch.float32).t()
    w = F.pad(w, (0, -k % BLOCK, 0, -m % BLOCK))
    tiles = w.view(w.shape[0] // BLOCK, BLOCK, w.shape[1] // BLOCK, BLOCK)
    e = _exponent(tiles.abs().amax(dim=(1, 3)))
    tiles = tiles * _power(-e).view(e.shape[0], 1, e.shape[1], 1)
    values = tiles.reshape(w.shape)[:m].to(torch.float8_e4m3fn).contiguous()
    return values, _as_scales(e)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = dict(case)
    if case["kind"] == "norm":
        dtype = DTYPES[case["dtype"]]
        s["x"] = _rows(gen, case["rows"], case["cols"], dtype)
        s["r"] = _rows(gen, case["rows"], case["cols"], dtype) if case["residual"] else None
        s["w"] = (1 + 0.2 * torch.randn(case["cols"], generator=gen, device=DEV)).to(dtype)
        if case["form"] == "grad":
            s["gy"] = _rows(gen, case["rows"], case["cols"], dtype, scale=0.01)
    elif case["kind"] == "fp8":
        if case["form"] == "linear":      # rows as the layer before leaves them
            s["x"] = _rows(gen, case["rows"], case["k"], torch.bfloat16, spread=1.0)
            s["w"] = _weight_8bit(gen, case["k"], case["m"])
        else:                             # rows as the norm leaves them
            s["x8"] = _quantize(_rows(gen, case["rows"], case["k"], torch.float32, spread=1.0))
            s["wg"] = _weight_8bit(gen, case["k"], case["m"])
            s["wu"] = _weight_8bit(gen, case["k"], case["m"])
    else:
        dtype = DTYPES[case["dtype"]]
        s["x"] = _rows(gen, case["rows"], case["k"], dtype, spread=0.2)
        s["wg"] = _weight(gen, case["k"], case["m"], dtype)
        s["wu"] = _weight(gen, case["k"], case["m"], dtype)
        if case["form"] == "grad":
            s["gh"] = _rows(gen, case["rows"], case["m"], dtype, spread=0.2, scale=0.01)
    return s


# ---- the plain forms -----------------------------------------------------------------------------

def _power(e):
    """2 to the whole numbers e in [-126, 126], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(amax):
    """Of the smallest power of two s with amax <= 448 s (448 = 0.875 * 2^9); 0 for blocks of zeros."""
    mantissa, exponent = torch.frexp(amax)
    e = (exponent - 9 + (mantissa > 0.875).int()).clamp(-126, 126)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _as_scales(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _of_scales(scales):
    return (scales.view(torch.uint8).int() << 23).view(torch.float32)


def _quantize(x):
    x = F.pad(x, (0, -x.shape[1] % BLOCK))
    blocks = x.view(x.shape[0], -1, BLOCK)
    e = _exponent(blocks.abs().amax(dim=2))
    values = (blocks * _power(-e).unsqueeze(2)).to(torch.float8_e4m3fn)
    return values.view(x.shape), _as_scales(e)


def _rows_of(x8, scales):
    return (x8.float().view(x8.shape[0], -1, BLOCK) * _of_scales(scales).unsqueeze(2)).view(x8.shape)


def _weight_of(w8, scales):
    s = _of_scales(scales).repeat_interleave(BLOCK, 0)[:w8.shape[0]]
    return (w8.float().view(w8.shape[0], -1, BLOCK) * s.unsqueeze(2)).view(w8.shape)


def _act(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return torch.clamp(g, min=0)


def _act_slope(name, g):
    if name == "silu":
        p = torch.sigmoid(g)
        return p * (1 + g * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return (g > 0).to(g.dtype)


def _plain_norm(s):
    x = s["x"].float()
    total = x if s["r"] is None else x + s["r"].float()
    inv = torch.rsqrt((total * total).mean(dim=1, keepdim=True) + EPS)
    w = s["w"].float()
    out = {}
    if s["form"] == "grad":       # the sum was kept by the forward pass: s["x"] is that sum here
        gy = s["gy"].float()
        wide = gy * w
        dot = (wide * x).mean(dim=1, keepdim=True)
        inv = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)
        gx = inv * wide - x * (inv * inv * inv * dot)
        if s["r"] is not None:
            gx = gx + s["r"].float()
        return {"grad_x": gx.to(s["x"].dtype), "grad_weight": (gy * x * inv).sum(dim=0).to(s["w"].dtype)}
    y = total * inv * w
    if s["form"] == "fp8":
        out["y8"], out["scales"] = _quantize(y)
    else:
        out["y"] = y.to(s["x"].dtype)
    if s["r"] is not None:
        out["sum"] = total.to(s["x"].dtype)
    return out


def _plain_fp8(s):
    if s["form"] == "linear":
        x = _rows_of(*_quantize(s["x"].float()))
        return torch.mm(x, _weight_of(*s["w"]).t()).to(torch.bfloat16)
    x = _rows_of(*s["x8"])
    gate = torch.mm(x, _weight_of(*s["wg"]).t())
    up = torch.mm(x, _weight_of(*s["wu"]).t())
    return (_act("silu", gate) * up).to(torch.bfloat16)


def _plain_gated(s):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    gate, up = torch.mm(x, wg), torch.mm(x, wu)
    if s["form"] == "forward":
        return (_act(s["act"], gate) * up).to(s["x"].dtype)
    gh = s["gh"].float()
    d_up = gh * _act(s["act"], gate)
    d_gate = gh * up * _act_slope(s["act"], gate)
    gx = torch.mm(d_gate, wg.t()) + torch.mm(d_up, wu.t())
    return {"grad_x": gx.to(s["x"].dtype), "grad_gate": torch.mm(x.t(), d_gate).to(s["x"].dtype),
            "grad_up": torch.mm(x.t(), d_up).to(s["x"].dtype)}


# ---- the framework's operators -------------------------------------------------------------------

def _own_norm(s):
    from graphiler_amd import ops
    if s["form"] == "grad":
        gx, gw = ops.rms_norm_backward(s["gy"], s["x"], s["w"], eps=EPS, grad_sum=s["r"])
        return {"grad_x": gx, "grad_weight": gw}
    if s["form"] == "fp8":
        got = ops.rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=EPS)
        names = ("y8", "scales", "sum")
    else:
        got = ops.rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
        names = ("y", "sum")
        got = got if s["r"] is not None else (got,)
    return dict(zip(names, got))


def _own_fp8(s):
    from graphiler_amd import ops
    if s["form"] == "linear":
        return ops.linear_fp8(*ops.quantize_fp8(s["x"]), *s["w"])
    return ops.gated_linear_fp8(*s["x8"], *s["wg"], *s["wu"], activation="silu")


def _own_gated(s):
    from graphiler_amd import ops
    if s["form"] == "forward":
        return ops.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"])
    got = ops.gated_linear_backward(s["gh"], s["x"], s["wg"], s["wu"], activation=s["act"])
    return dict(zip(("grad_x", "grad_gate", "grad_up"), got))


def run(state):
    kind = state["kind"]
    if own:
        return _own_norm(state) if kind == "norm" else _own_fp8(state) if kind == "fp8" else _own_gated(state)
    return _plain_norm(state) if kind == "norm" else _plain_fp8(state) if kind == "fp8" else _plain_gated(state)


# ---- the definition in 64 bits -------------------------------------------------------------------

_ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def _wide(values, scales, rows_each):
    """8-bit values times their scales, the exponents read from the scales' own bits."""
    e = scales.view(torch.uint8).double() - 127
    e = torch.repeat_interleave(torch.repeat_interleave(e, rows_each, 0)[:values.shape[0]], BLOCK, 1)
    return values.double() * torch.pow(torch.full_like(e, 2.0), e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        x, w = s["x"].double(), s["w"].double()
        if case["form"] == "grad":
            x.requires_grad_(), w.requires_grad_()
            y = x / (x.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w
            gx, gw = torch.autograd.grad(y, (x, w), s["gy"].double())
            return {"grad_x": gx if s["r"] is None else gx + s["r"].double(), "grad_weight": gw}
        total = x if s["r"] is None else x + s["r"].double()
        y = total / (total.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w
        out = {"y": y}
        if case["form"] == "fp8":         # the values before they are cut to 8 bits, and the scales
            n = -(-case["cols"] // BLOCK)
            padded = torch.zeros(case["rows"], n * BLOCK, dtype=torch.float64, device=DEV)
            padded[:, :case["cols"]] = y
            blocks = padded.view(case["rows"], n, BLOCK)
            scale = torch.pow(2.0, torch.ceil(torch.log2(blocks.abs().amax(2) / 448).clamp(min=-126)))
            out = {"y8": (blocks / scale.unsqueeze(2)).view_as(padded), "scales": scale}
        if s["r"] is not None:
            out["sum"] = total
        return out
    if case["kind"] == "fp8":
        if case["form"] == "linear":
            return _wide(*_quantize(s["x"].float()), 1) @ _wide(*s["w"], BLOCK).T
        x = _wide(*s["x8"], 1)
        return F.silu(x @ _wide(*s["wg"], BLOCK).T) * (x @ _wide(*s["wu"], BLOCK).T)
    args = [s[k].double().requires_grad_(case["form"] == "grad") for k in ("x", "wg", "wu")]
    h = _ACTS[case["act"]](args[0] @ args[1]) * (args[0] @ args[2])
    if case["form"] == "forward":
        return h
    return dict(zip(("grad_x", "grad_gate", "grad_up"), torch.autograd.grad(h, args, s["gh"].double())))


# ---- what a pass has to move and compute ---------------------------------------------------------

def work(case):
    rows = case["rows"]
    if case["kind"] == "norm":
        cols, size = case["cols"], BYTES[case["dtype"]]
        blocks = -(-cols // BLOCK)
        n = rows * cols * size
        if case["form"] == "grad":        # the sum, its gradient and the gradient of y read, that of x written
            return {"bytes": n * (4 if case["residual"] else 3) + 2 * cols * size, "flops": 9 * rows * cols}
        out = rows * blocks * (BLOCK + 1) if case["form"] == "fp8" else n
        return {"bytes": n + out + (2 * n if case["residual"] else 0) + cols * size, "flops": 5 * rows * cols}
    if case["kind"] == "fp8":
        k, m = -(-case["k"] // BLOCK) * BLOCK, case["m"]
        weights = 2 if case["form"] == "gated" else 1
        x = rows * k * (1 + 1 / BLOCK) if case["form"] == "gated" else rows * case["k"] * 2
        w = weights * (m * k + -(-m // BLOCK) * (k // BLOCK))
        return {"bytes": x + w + rows * m * 2, "flops": 2 * rows * case["k"] * m * weights}
    k, m, size = case["k"], case["m"], BYTES[case["dtype"]]
    product = 2 * rows * k * m
    if case["form"] == "forward":
        return {"bytes": (rows * k + 2 * k * m + rows * m) * size, "flops": 2 * product}
    # both projections again, the gradient of the rows, the gradients of both weights
    return {"bytes": (2 * rows * k + 4 * k * m + rows * m) * size, "flops": 6 * product}
