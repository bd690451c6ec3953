"""What a transformer over graphs adds to the layers along edges, as cases that can be timed: attention
inside every segment of packed rows (a graph's nodes, a sequence of them) with its gradients, the
projections around it with bias, activation and residual, and the embedding rows that it begins with.

A case is one call, or a forward and a backward call, as a user's program makes them (with ``own``: the
framework's operators; without: the same definition in elementary torch operations, in 32 bits,
rounded once at the end).

Attention: query i of a segment sees the keys of its segment, with ``causal`` those at positions
j <= i + (keys - queries); a query that sees none gives zeros, as do rows behind the last segment.
Embedding: an id outside the table gives zeros and receives nothing.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "bf16": 2}


def listed():
    return [
        # One molecule is answered by itself: the smallest call, its latency counts.
        {"name": "attention_one_molecule", "kind": "attention", "form": "forward", "segments": 1, "queries": 29,
         "keys": 0, "heads": 4, "groups": 1, "dim": 16, "causal": False, "dtype": "bf16", "spare": 0},
        # Training on a batch of molecules, 9 to 60 nodes each, hidden width 256: many short segments.
        {"name": "attention_molecules_train", "kind": "attention", "form": "train", "segments": 2_048, "queries": 60,
         "keys": 0, "heads": 8, "groups": 1, "dim": 32, "causal": False, "dtype": "bf16", "spare": 0},
        # Every node of a citation graph attends to every other, the benchmark's width of 64 a head.
        {"name": "attention_all_nodes", "kind": "attention", "form": "forward", "segments": 1, "queries": 19_717,
         "keys": 0, "heads": 8, "groups": 1, "dim": 64, "causal": False, "dtype": "bf16", "spare": 0},
        # Node sequences in order (prompts): causal, four query heads share a key head, lengths apart.
        {"name": "attention_sequences", "kind": "attention", "form": "forward", "segments": 4, "queries": 4_096,
         "keys": 0, "heads": 16, "groups": 4, "dim": 128, "causal": True, "dtype": "bf16", "spare": 0},
        # Training on such sequences.
        {"name": "attention_sequences_train", "kind": "attention", "form": "train", "segments": 4, "queries": 4_096,
         "keys": 0, "heads": 16, "groups": 4, "dim": 128, "causal": True, "dtype": "bf16", "spare": 0},
        # Training in fp32 on subgraphs of a citation graph, heads of a width that no tile has.
        {"name": "attention_fp32_train", "kind": "attention", "form": "train", "segments": 5, "queries": 683,
         "keys": 0, "heads": 3, "groups": 1, "dim": 20, "causal": False, "dtype": "fp32", "spare": 7},
        # Serving, and the readout of large graphs: one new query for each over all it has so far.
        {"name": "attention_one_query_each", "kind": "attention", "form": "forward", "segments": 16, "queries": 1,
         "keys": 16_384, "heads": 32, "groups": 8, "dim": 128, "causal": True, "dtype": "bf16", "spare": 0},
        # Three nodes are answered together: the projection behind their attention, onto the stream.
        {"name": "linear_three_rows", "kind": "linear", "form": "forward", "rows": 3, "k": 1_024, "m": 4_096,
         "dtype": "bf16", "act": "gelu", "bias": True, "residual": True},
        # A citation graph's 500 input features to the hidden width in fp32.
        {"name": "linear_nodes_fp32", "kind": "linear", "form": "forward", "rows": 19_717, "k": 500, "m": 256,
         "dtype": "fp32", "act": "relu", "bias": True, "residual": False},
        # Training of a wide block's first projection.
        {"name": "linear_train", "kind": "linear", "form": "grad", "rows": 8_192, "k": 1_024, "m": 4_096,
         "dtype": "bf16", "act": "gelu", "bias": True, "residual": True},
        # The rows that nodes begin with, a table of as many rows as a vocabulary has, some ids often.
        {"name": "embedding_nodes", "kind": "embedding", "form": "forward", "rows": 262_144, "table": 32_000,
         "cols": 512, "dtype": "bf16", "skew": 3.0},
        # Training of that table: sums over the rows of every id.
        {"name": "embedding_train", "kind": "embedding", "form": "grad", "rows": 65_536, "table": 32_000,
         "cols": 1_024, "dtype": "bf16", "skew": 3.0},
    ]


# most of what a pass of a drawn case may compute or move
MOST_PAIRS = 8 * 19_717 * 19_717
MOST_FLOPS = {"attention": {"bf16": 1.1e12, "fp32": 4e10}, "linear": {"bf16": 4.1e11, "fp32": 4e10}}
MOST_VALUES = 262_144 * 512


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """Half of the widths are multiples of 64, the others any number."""
    if rng.random() < 0.5:
        return max(low, min(high, _spread(rng, max(low, 64), high) // 64 * 64))
    return _spread(rng, low, high)


def draw(rng):
    while True:
        kind = rng.choice(["attention", "attention", "linear", "embedding"])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        if kind == "attention":
            form, few = rng.choice(["forward", "train"]), rng.random() < 0.3
            groups, kv_heads = rng.choice([1, 1, 2, 4, 8]), _spread(rng, 1, 8)
            case = {"kind": kind, "form": "forward" if few else form,
                    "segments": _spread(rng, 1, 64 if few else 2_048),
                    "queries": _spread(rng, 1, 4) if few else _spread(rng, 1, 8_192),
                    "keys": _spread(rng, 64, 32_768) if few else rng.choice([0, 0, 0, _spread(rng, 1, 8_192)]),
                    "heads": groups * kv_heads, "groups": groups,
                    "dim": rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, rng.randint(1, 128)]),
                    "causal": rng.random() < 0.5, "dtype": dtype, "spare": rng.choice([0, 0, rng.randint(1, 40)])}
            keys = case["keys"] or case["queries"]
            if case["segments"] * case["heads"] * case["queries"] * keys <= MOST_PAIRS and \
                    case["segments"] * keys * case["heads"] * case["dim"] <= 2 * MOST_VALUES and \
                    work(case)["flops"] <= MOST_FLOPS[kind][dtype]:
                return case
        elif kind == "linear":
            case = {"kind": kind, "form": rng.choice(["forward", "grad"]), "rows": _spread(rng, 1, 65_536),
                    "k": _width(rng, 16, 4_096), "m": _width(rng, 16, 8_192), "dtype": dtype,
                    "act": rng.choice(["none", "silu", "gelu", "relu"]), "bias": rng.random() < 0.7,
                    "residual": rng.random() < 0.5}
            if work(case)["flops"] <= MOST_FLOPS[kind][dtype] and case["rows"] * case["m"] <= MOST_VALUES:
                return case
        else:
            case = {"kind": kind, "form": rng.choice(["forward", "grad"]), "rows": _spread(rng, 1, 524_288),
                    "table": _spread(rng, 2, 131_072), "cols": _width(rng, 16, 2_048), "dtype": dtype,
                    "skew": rng.choice([1.0, 2.0, 4.0])}
            if max(case["rows"], case["table"]) * case["cols"] * BYTES[dtype] <= 2 * MOST_VALUES:
                return case


# ---- inputs --------------------------------------------------------------------------------------

def _lengths(segments, most):
    """Lengths from a seventh of the longest on, the longest first, spread evenly and out of order."""
    low = -(-most // 7)
    return [most - int((most - low) * (i * 0.6180339887498949 % 1.0)) for i in range(segments)]


def _case_lengths(case):
    q = _lengths(case["segments"], case["queries"])
    if case["keys"] == 0:
        return q, q
    return q, list(reversed(_lengths(case["segments"], case["keys"])))


def _pairs(case):
    """Pairs of a query and a key that it sees, of one head."""
    n = 0
    for a, b in zip(*_case_lengths(case)):
        if not case["causal"]:
            n += a * b
        elif b >= a:                  # query i sees i + 1 + (b - a) keys
            n += a * (b - a) + a * (a + 1) // 2
        else:                         # the first a - b see none
            n += b * (b + 1) // 2
    return n


def _rows(gen, rows, cols, dtype, spread=0.2, scale=1.0):
    """Normal values whose columns differ in size, as the features of a trained network do."""
    width = torch.exp(spread * torch.randn(cols, generator=gen, device=DEV))
    return torch.randn(rows, cols, generator=gen, device=DEV).mul_(width).mul_(scale).to(dtype)


def _pointer(lengths):
    p = [0]
    for n in lengths:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s, dtype = dict(case), DTYPES[case["dtype"]]
    if case["kind"] == "attention":
        heads, dim = case["heads"], case["dim"]
        kv = heads // case["groups"]
        nq, nk = (sum(n) + case["spare"] for n in _case_lengths(case))
        s["qp"], s["kp"] = (_pointer(n) for n in _case_lengths(case))
        # keys and values (and queries of the same rows) are columns of one projection's result
        if case["keys"] == 0:
            rows = _rows(gen, nq, (heads + 2 * kv) * dim, dtype)
            rows[:, :heads * dim] *= 1.5
            s["q"] = rows[:, :heads * dim].view(nq, heads, dim)
            rows = rows[:, heads * dim:]
            s["kp"] = s["qp"]
        else:
            s["q"] = _rows(gen, nq, heads * dim, dtype, scale=1.5).view(nq, heads, dim)
            rows = _rows(gen, nk, 2 * kv * dim, dtype)
        s["k"] = rows[:, :kv * dim].view(nk, kv, dim)
        s["v"] = rows[:, kv * dim:].view(nk, kv, dim)
        if case["form"] == "train":
            s["go"] = _rows(gen, nq, heads * dim, dtype, scale=0.01).view(nq, heads, dim)
    elif case["kind"] == "linear":
        s["x"] = _rows(gen, case["rows"], case["k"], dtype)
        s["w"] = (torch.randn(case["k"], case["m"], generator=gen, device=DEV) / math.sqrt(case["k"])).to(dtype)
        s["b"] = _rows(gen, 1, case["m"], dtype, scale=0.5)[0] if case["bias"] else None
        s["r"] = _rows(gen, case["rows"], case["m"], dtype) if case["residual"] else None
        if case["form"] == "grad":
            s["gy"] = _rows(gen, case["rows"], case["m"], dtype, scale=0.01)
    else:
        at = torch.rand(case["rows"], generator=gen, device=DEV, dtype=torch.float64)
        s["ids"] = (at.pow(case["skew"]) * case["table"]).long().clamp(max=case["table"] - 1)
        s["ids"][torch.rand(case["rows"], generator=gen, device=DEV) < 0.02] = -1        # padding
        s["scale"] = math.sqrt(case["cols"])
        if case["form"] == "grad":
            s["gy"] = _rows(gen, case["rows"], case["cols"], dtype, scale=0.01)
        else:
            s["t"] = _rows(gen, case["table"], case["cols"], dtype, scale=case["cols"] ** -0.5)
    return s


# ---- the plain forms -----------------------------------------------------------------------------

def _act(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return torch.clamp(z, min=0) if name == "relu" else z


def _act_slope(name, z):
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return (z > 0).to(z.dtype) if name == "relu" else torch.ones_like(z)


def _padded(x, pointer, longest):
    """(segments, heads, longest, dim) fp32 of packed rows; which of them there are."""
    at = torch.arange(longest, device=DEV)
    there = at < (pointer[1:] - pointer[:-1]).unsqueeze(1)
    rows = (pointer[:-1].unsqueeze(1) + at).clamp(max=x.shape[0] - 1)
    padded = x[rows].float() * there.view(*there.shape, 1, 1)
    return padded.transpose(1, 2).contiguous(), there


def _packed(padded, pointer, there, rows, dtype):
    """The rows of a padded tensor where they lie in the packed one; zeros behind them."""
    out = torch.zeros(rows, padded.shape[1], padded.shape[3], dtype=dtype, device=DEV)
    found = padded.transpose(1, 2)[there].to(dtype)
    out[:found.shape[0]] = found
    return out


def _plain_attention(s):
    dtype, scale, groups = s["q"].dtype, 1.0 / math.sqrt(s["dim"]), s["groups"]
    longest_q, longest_k = s["queries"], s["keys"] or s["queries"]
    q, q_there = _padded(s["q"], s["qp"], longest_q)
    k, k_there = _padded(s["k"], s["kp"], longest_k)
    v, _ = _padded(s["v"], s["kp"], longest_k)
    b, kv, d = q.shape[0], k.shape[1], s["dim"]
    by_head = (b * kv, groups * longest_q, longest_k)
    flat = lambda x: x.reshape(b * kv, -1, d)          # noqa: E731  (the heads of a group, one behind the other)
    seen = k_there.view(b, 1, longest_k).expand(b, longest_q, longest_k)
    if s["causal"]:
        more = (s["kp"].diff() - s["qp"].diff()).view(b, 1, 1)
        i = torch.arange(longest_q, device=DEV).view(1, -1, 1)
        seen = seen & (torch.arange(longest_k, device=DEV) <= i + more)
    seen = seen.view(b, 1, 1, longest_q, longest_k)
    p = torch.bmm(flat(q), flat(k).transpose(1, 2)).mul_(scale).view(b, kv, groups, longest_q, longest_k)
    p = p.masked_fill_(~seen, -math.inf)
    most = p.amax(dim=-1, keepdim=True)
    p = p.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total))).view(by_head)
    out = torch.bmm(p, flat(v))
    result = _packed(out.view(b, kv * groups, longest_q, d), s["qp"], q_there, s["q"].shape[0], dtype)
    if s["form"] == "forward":
        return result
    go = flat(_padded(s["go"], s["qp"], longest_q)[0])
    grad_v = torch.bmm(p.transpose(1, 2), go)
    ds = torch.bmm(go, flat(v).transpose(1, 2)).sub_((go * out).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    grad_q, grad_k = torch.bmm(ds, flat(k)), torch.bmm(ds.transpose(1, 2), flat(q))
    of_keys = lambda g: _packed(g.view(b, kv, longest_k, d), s["kp"], k_there, s["k"].shape[0], dtype)  # noqa: E731
    return {"out": result, "grad_k": of_keys(grad_k), "grad_v": of_keys(grad_v),
            "grad_q": _packed(grad_q.view(b, kv * groups, longest_q, d), s["qp"], q_there, s["q"].shape[0], dtype)}


def _plain_linear(s):
    x, w, dtype = s["x"].float(), s["w"].float(), s["x"].dtype
    if s["form"] == "forward" or s["act"] != "none":
        z = torch.mm(x, w)
        if s["b"] is not None:
            z = z + s["b"].float()
    if s["form"] == "forward":
        y = _act(s["act"], z)
        return (y if s["r"] is None else y + s["r"].float()).to(dtype)
    dz = s["gy"].float()
    if s["act"] != "none":
        dz = dz * _act_slope(s["act"], z)
    out = {"grad_x": torch.mm(dz, w.t()).to(dtype), "grad_w": torch.mm(x.t(), dz).to(dtype)}
    if s["b"] is not None:
        out["grad_b"] = dz.sum(dim=0).to(dtype)
    return out


def _plain_embedding(s):
    ids = s["ids"]
    there = ((ids >= 0) & (ids < s["table"])).unsqueeze(1)
    ids = ids.clamp(0, s["table"] - 1)
    if s["form"] == "forward":
        return (s["t"][ids].float() * there * s["scale"]).to(s["t"].dtype)
    grad = torch.zeros(s["table"], s["cols"], dtype=torch.float32, device=DEV)
    grad.index_add_(0, ids, s["gy"].float() * there)
    return (grad * s["scale"]).to(s["gy"].dtype)


# ---- the framework's operators -------------------------------------------------------------------

def _own_attention(s):
    from graphiler_amd import ops
    if s["form"] == "forward":
        return ops.segment_attention(s["q"], s["k"], s["v"], s["qp"], s["kp"], causal=s["causal"])
    out, lse = ops.segment_attention(s["q"], s["k"], s["v"], s["qp"], s["kp"], causal=s["causal"], return_lse=True)
    gq, gk, gv = ops.segment_attention_backward(s["go"], s["q"], s["k"], s["v"], out, lse, s["qp"], s["kp"],
                                                causal=s["causal"])
    return {"out": out, "grad_q": gq, "grad_k": gk, "grad_v": gv}


def _own_linear(s):
    from graphiler_amd import ops
    act = None if s["act"] == "none" else s["act"]
    if s["form"] == "forward":
        return ops.linear_act(s["x"], s["w"], bias=s["b"], activation=act, residual=s["r"])
    gx, gw, gb = ops.linear_act_backward(s["gy"], s["x"], s["w"], bias=s["b"], activation=act)
    return {"grad_x": gx, "grad_w": gw} if gb is None else {"grad_x": gx, "grad_w": gw, "grad_b": gb}


def _own_embedding(s):
    from graphiler_amd import ops
    if s["form"] == "forward":
        return ops.embedding(s["t"], s["ids"], scale=s["scale"])
    return ops.embedding_backward(s["gy"], s["ids"], s["table"], scale=s["scale"])


def run(state):
    kind = state["kind"]
    if own:
        return _own_attention(state) if kind == "attention" else _own_linear(state) if kind == "linear" \
            else _own_embedding(state)
    return _plain_attention(state) if kind == "attention" else _plain_linear(state) if kind == "linear" \
        else _plain_embedding(state)


# ---- the definition in 64 bits -------------------------------------------------------------------

def _exact_attention(case, s):
    train, groups = case["form"] == "train", case["groups"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    out, grads = torch.zeros_like(q), [torch.zeros_like(t) for t in (q, k, v)]
    a = c = 0
    for n, m in zip(*_case_lengths(case)):
        # a head at a time where all would not fit, all of a short segment's at once
        for heads in ([range(k.shape[1])] if n * m < 1 << 20 else [[h] for h in range(k.shape[1])]):
            kh = list(heads)
            qh = [h * groups + g for h in kh for g in range(groups)]
            x, y, z = q[a:a + n, qh].transpose(0, 1), k[c:c + m, kh].transpose(0, 1), v[c:c + m, kh].transpose(0, 1)
            parts = [t.contiguous().requires_grad_(train) for t in (x, y, z)]
            y, z = (t.repeat_interleave(groups, 0) for t in parts[1:])
            scores = parts[0] @ y.transpose(1, 2).contiguous() / math.sqrt(case["dim"])
            if case["causal"]:
                seen = torch.ones(n, m, dtype=torch.bool, device=DEV).tril(m - n)
                weights = torch.softmax(scores.masked_fill(~seen, -1e300), -1) * seen
            else:
                weights = torch.softmax(scores, -1)
            o = weights @ z.contiguous()
            out[a:a + n, qh] = o.detach().transpose(0, 1)
            if train:
                found = torch.autograd.grad(o, parts, s["go"][a:a + n, qh].double().transpose(0, 1).contiguous())
                grads[0][a:a + n, qh] = found[0].transpose(0, 1)
                grads[1][c:c + m, kh] = found[1].transpose(0, 1)
                grads[2][c:c + m, kh] = found[2].transpose(0, 1)
        a, c = a + n, c + m
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]} if train else out


_ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "none": lambda z: z}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    if case["kind"] == "embedding":
        if case["form"] == "forward":
            rows = torch.cat([s["t"].double(), torch.zeros(1, case["cols"], dtype=torch.float64, device=DEV)])
            return rows[torch.where(s["ids"] < 0, case["table"], s["ids"])] * s["scale"]
        order = torch.sort(s["ids"], stable=True)
        sums = torch.zeros(case["table"] + 1, case["cols"], dtype=torch.float64, device=DEV)
        sums.index_put_((order.values + 1,), s["gy"].double()[order.indices], accumulate=True)
        return sums[1:] * s["scale"]
    names = [n for n in ("x", "w", "b") if s[n] is not None]
    args = {n: s[n].double().requires_grad_(case["form"] == "grad") for n in names}
    z = args["x"] @ args["w"]
    y = _ACTS[case["act"]](z + args["b"] if "b" in args else z)
    if case["form"] == "forward":
        return y if s["r"] is None else y + s["r"].double()
    return dict(zip(("grad_" + n for n in names), torch.autograd.grad(y, [args[n] for n in names], s["gy"].double())))


# ---- what a pass has to move and compute ---------------------------------------------------------

def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "attention":
        q, k = (sum(n) for n in _case_lengths(case))
        q, k = q * case["heads"] * case["dim"] * size, k * case["heads"] // case["groups"] * case["dim"] * size
        pair = 4 * case["dim"] * case["heads"] * _pairs(case)
        if case["form"] == "forward":     # q, k, v read, the result written; two products
            return {"bytes": 2 * q + 2 * k, "flops": pair}
        # and its gradient read, three gradients written; five products more
        return {"bytes": 4 * q + 4 * k, "flops": 3.5 * pair}
    rows = case["rows"]
    if case["kind"] == "linear":
        k, m = case["k"], case["m"]
        product = 2 * rows * k * m
        if case["form"] == "forward":
            more = rows * m if case["residual"] else 0
            return {"bytes": (rows * k + k * m + rows * m + more) * size, "flops": product}
        # the product again where an activation's slope needs it, the gradients of the rows and of the weight
        return {"bytes": (2 * rows * k + 2 * k * m + rows * m) * size,
                "flops": (2 if case["act"] == "none" else 3) * product}
    cols, table = case["cols"], case["table"]
    if case["form"] == "forward":         # rows of the table at most once each
        return {"bytes": rows * 8 + (rows + min(rows, table)) * cols * size, "flops": rows * cols}
    return {"bytes": rows * 8 + (rows + table) * cols * size, "flops": rows * cols}
