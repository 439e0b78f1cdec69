"""Attention over packed records and the orthogonalised optimizer step, as measurable cases.

Two parts of a LoRA training step next to the projections: the decoder's attention (the
forward, the backward that recomputes the probabilities, and the form in which a few query
tokens read a long key/value cache), and the Muon update of the adapters (momentum, a
Newton-Schulz iteration towards the nearest orthogonal matrix, the parameter update).
With `own` false every case is computed by elementary torch operations in 32 bits.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MUON = {"lr": 2e-2, "momentum": 0.95, "weight_decay": 0.1}

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "causal-tuner_amd"))


def listed():
    return [
        # One answer being written: one token of a 16-head decoder against a short cache. Latency.
        {"name": "attention-token", "kind": "attention", "direction": "forward", "queries": "1", "keys": "700",
         "heads": 16, "kv_heads": 1, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # A batch of answers at different lengths, one token each, grouped heads.
        {"name": "attention-token-batch", "kind": "attention", "direction": "forward",
         "queries": ",".join(["1"] * 24),
         "keys": "311,9001,4096,2047,1,640,5555,1203,77,8192,3001,129,700,6400,2500,911,4800,64,1777,7000,350,1024,33,5120",
         "heads": 32, "kv_heads": 8, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # One token against a very long cache: the stream of keys and values is the work.
        {"name": "attention-token-long", "kind": "attention", "direction": "forward", "queries": "1",
         "keys": "131072", "heads": 32, "kv_heads": 8, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # Evaluation of two prompts, one of which continues 4000 cached tokens.
        {"name": "attention-prompt", "kind": "attention", "direction": "forward", "queries": "1000,37",
         "keys": "5000,37", "heads": 16, "kv_heads": 1, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # The training step of a decoder layer over three packed records.
        {"name": "attention-train-records", "kind": "attention", "direction": "train", "queries": "1411,806,1204",
         "keys": "1411,806,1204", "heads": 16, "kv_heads": 1, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # One long record of a 4096-wide layer: the largest matrix products.
        {"name": "attention-train-long", "kind": "attention", "direction": "train", "queries": "8192",
         "keys": "8192", "heads": 32, "kv_heads": 1, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # Ragged records seen in both directions, grouped heads of 64.
        {"name": "attention-train-ragged", "kind": "attention", "direction": "train", "queries": "1,129,640,77,2001",
         "keys": "1,129,640,77,2001", "heads": 12, "kv_heads": 4, "head_dim": 64, "causal": False, "dtype": "bf16"},
        # The float32 compute dtype.
        {"name": "attention-train-float32", "kind": "attention", "direction": "train", "queries": "333,500",
         "keys": "333,500", "heads": 8, "kv_heads": 1, "head_dim": 64, "causal": True, "dtype": "f32"},
        # The adapter of one small projection (rank 16): launches and latency.
        {"name": "orthogonalize-small", "kind": "orthogonalize", "shapes": "16x1024,1024x16", "dtype": "f32"},
        # Half-width gradients of odd shapes, wide and tall.
        {"name": "orthogonalize-odd", "kind": "orthogonalize", "shapes": "130x1111,2049x64,255x257,8x3001,4100x128",
         "dtype": "bf16"},
        # The optimizer step of one layer's adapters (d 2048, inner 8192, rank 256).
        {"name": "muon-layer", "kind": "muon", "layers": 1, "inputs": 2048, "inner": 8192, "rank": 256,
         "dtype": "f32"},
        # The optimizer step of two wide layers' adapters (d 4096, inner 11008, rank 256).
        {"name": "muon-two-layers", "kind": "muon", "layers": 2, "inputs": 4096, "inner": 11008, "rank": 256,
         "dtype": "f32"},
    ]


# ----------------------------------------------------------------------------- drawing cases
def _between(rng, low, high):
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["token", "prompt", "train", "train", "train", "orthogonalize", "muon"])
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw_kind(rng, kind)
        cost = work(case)
        if cost["flops"] <= 0.7 * most["flops"] and cost["bytes"] <= 0.7 * most["bytes"]:
            return case


def _draw_kind(rng, kind):
    if kind == "orthogonalize":
        shapes = []
        for _ in range(rng.randint(1, 12)):
            short, long = _between(rng, 1, 300), _between(rng, 16, 8192)
            shapes.append("%dx%d" % ((short, long) if rng.random() < 0.5 else (long, short)))
        return {"kind": kind, "shapes": ",".join(shapes), "dtype": rng.choice(["f32", "f32", "bf16"])}
    if kind == "muon":
        return {"kind": kind, "layers": rng.randint(1, 2), "inputs": _between(rng, 8, 64) * 64,
                "inner": _between(rng, 16, 172) * 64, "rank": rng.choice([8, 16, 32, 64, 128, 256, 256]),
                "dtype": rng.choice(["f32", "f32", "f32", "bf16"])}
    kv_heads = rng.choice([1, 1, 1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8] if kv_heads > 1 else [1, 4, 8, 12, 16, 24, 32])
    case = {"kind": "attention", "direction": "forward", "heads": heads, "kv_heads": kv_heads,
            "head_dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128]), "causal": rng.random() < 0.85,
            "dtype": "f32" if rng.random() < 0.2 else "bf16"}
    top = 1024 if case["dtype"] == "f32" else 4096
    if kind == "token":
        keys = [_between(rng, 1, 32768) for _ in range(_between(rng, 1, 32))]
        queries = [1 if rng.random() < 0.9 else min(k, rng.randint(1, 4)) for k in keys]
    elif kind == "prompt":
        queries = [_between(rng, 2, top) for _ in range(rng.randint(1, 3))]
        keys = [q + (_between(rng, 1, top) if rng.random() < 0.6 else 0) for q in queries]
    else:
        case["direction"] = "train"
        keys = queries = [_between(rng, 1, top) for _ in range(rng.randint(1, 4))]
    return {**case, "queries": ",".join(map(str, queries)), "keys": ",".join(map(str, keys))}


# ----------------------------------------------------------------------------- inputs
def _sizes(text):
    return [int(n) for n in text.split(",")]


def _records(sizes):
    bounds, start = [], 0
    for size in sizes:
        bounds.append((start, start + size))
        start += size
    return bounds


def _adapter_shapes(case):
    """A and B of q, k, v, o, gate, up and down, layer by layer."""
    d, inner, r = case["inputs"], case["inner"], case["rank"]
    pairs = [(d, d), (d, 128), (d, 128), (d, d), (d, inner), (d, inner), (inner, d)]
    return [shape for _ in range(case["layers"]) for k, n in pairs for shape in ((r, k), (n, r))]


def _matrix_shapes(case):
    if case["kind"] == "muon":
        return _adapter_shapes(case)
    return [tuple(int(n) for n in text.split("x")) for text in case["shapes"].split(",")]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) & 0x7fffffffffffffff)


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=DEVICE, generator=g) * std).to(dtype)


def _gradient(g, shape, dtype):
    """A gradient as adapters meet it: a few strong directions over a flat background."""
    rows, cols = shape
    strong = min(rows, cols, 8)
    left, right = _normal(g, rows, strong, dtype=torch.float32), _normal(g, strong, cols, dtype=torch.float32)
    return ((left @ right) * 1e-3 + _normal(g, rows, cols, std=1e-3, dtype=torch.float32)).to(dtype)


def _padding(bounds, longest):
    """Row numbers [records, longest] (0 where a record is shorter) and the places, in the
    flattened padded layout, of all the rows in order."""
    rows = torch.zeros(len(bounds), longest, dtype=torch.int64)
    places = []
    for i, (start, stop) in enumerate(bounds):
        rows[i, :stop - start] = torch.arange(start, stop)
        places.append(torch.arange(stop - start) + i * longest)
    return rows.to(DEVICE), torch.cat(places).to(DEVICE)


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "attention":
        queries, keys = _records(_sizes(case["queries"])), _records(_sizes(case["keys"]))
        train = case["direction"] == "train"
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
        state.update(q=_normal(g, queries[-1][1], heads, dim, std=1.5, dtype=dtype).requires_grad_(train),
                     k=_normal(g, keys[-1][1], kv_heads, dim, dtype=dtype).requires_grad_(train),
                     v=_normal(g, keys[-1][1], kv_heads, dim, dtype=dtype).requires_grad_(train))
        if train:
            state["dy"] = _normal(g, queries[-1][1], heads, dim, dtype=dtype)
        if own:
            from causal_tuner.kernels.attention_cuda import AttentionLayout
            state["layout"] = AttentionLayout(queries, DEVICE, key_records=keys)
        else:
            # what the batch says of its own shape, made once where the batch is built
            lq, lk = (torch.tensor(_sizes(case[name]), device=DEVICE) for name in ("queries", "keys"))
            most_q, most_k = max(_sizes(case["queries"])), max(_sizes(case["keys"]))
            row, column = torch.arange(most_q, device=DEVICE), torch.arange(most_k, device=DEVICE)
            mask = (row[None, :, None] < lq[:, None, None]) & (column[None, None, :] < lk[:, None, None])
            if case["causal"]:
                mask &= column[None, None, :] <= row[None, :, None] + (lk - lq)[:, None, None]
            state.update(rows=_padding(queries, most_q), columns=_padding(keys, most_k), hidden=~mask[:, None, None])
        return state
    shapes = _matrix_shapes(case)
    gradients = [_gradient(g, shape, dtype) for shape in shapes]
    if case["kind"] == "orthogonalize":
        state["matrices"] = gradients
        return state
    params = [torch.nn.Parameter(_normal(g, *shape, std=0.02, dtype=dtype)) for shape in shapes]
    buffers = [_gradient(g, shape, torch.float32) * 0.5 for shape in shapes]
    for p, grad in zip(params, gradients):
        p.grad = grad
    state.update(params=params, buffers=buffers)
    if own:
        from causal_tuner.optim import FusedMuon
        state["optimizer"] = FusedMuon(params, **MUON)
        for p, buffer in zip(params, buffers):
            state["optimizer"].state[p]["momentum_buffer"] = buffer
    return state


# ----------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["kind"] == "attention":
        if not own:
            return _plain_attention(state)
        from causal_tuner.kernels.attention_cuda import packed_attention
        out = packed_attention(state["q"], state["k"], state["v"], state["layout"], causal=case["causal"])
        if case["direction"] == "forward":
            return out
        return (out, *torch.autograd.grad(out, [state["q"], state["k"], state["v"]], state["dy"]))
    if case["kind"] == "orthogonalize":
        if not own:
            return _plain_orthogonalize(state["matrices"])
        from causal_tuner.optim import orthogonalize
        return orthogonalize(state["matrices"])
    if not own:
        return _plain_muon(state)
    state["optimizer"].step()
    return tuple(state["params"]) + tuple(state["buffers"])


def _plain_attention(state):
    """softmax(q k^T / sqrt(d)) v over the records as one padded batch, the query heads of a
    key/value head side by side; with its gradients where the case trains."""
    case = state["case"]
    with torch.no_grad():
        q, k, v = state["q"], state["k"], state["v"]
        heads, dim = q.shape[1:]
        kv_heads = k.shape[1]
        (rows, row_places), (columns, column_places) = state["rows"], state["columns"]
        scale = 1 / math.sqrt(dim)

        def gather_rows(x):      # [tokens, heads, dim] -> [records, kv_heads, group * queries, dim]
            x = x.float()[rows].reshape(*rows.shape, kv_heads, heads // kv_heads, dim)
            return x.permute(0, 2, 3, 1, 4).reshape(len(rows), kv_heads, -1, dim)

        def gather_columns(x):   # [tokens, kv_heads, dim] -> [records, kv_heads, keys, dim]
            return x.float()[columns].transpose(1, 2).contiguous()

        def scatter_rows(x):
            x = x.reshape(len(rows), heads, rows.shape[1], dim).transpose(1, 2).reshape(-1, heads, dim)
            return x[row_places].to(q.dtype)

        def scatter_columns(x):
            return x.transpose(1, 2).reshape(-1, kv_heads, dim)[column_places].to(k.dtype)

        query, key, value = gather_rows(q), gather_columns(k), gather_columns(v)
        apart = (len(rows), kv_heads, heads // kv_heads, rows.shape[1], columns.shape[1])
        p = ((query @ key.transpose(2, 3)) * scale).view(apart).masked_fill_(state["hidden"], -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(top.masked_fill_(top == -math.inf, 0)).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(total.masked_fill_(total == 0, 1)).flatten(2, 3)
        out = p @ value
        if case["direction"] == "forward":
            return scatter_rows(out)
        dy = gather_rows(state["dy"])
        ds = (dy @ value.transpose(2, 3)).sub_((dy * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        # rows past a record's end are copies of row 0: they give nothing to the keys' gradients
        padded = state["hidden"].all(-1).expand(apart[:-1]).flatten(2, 3)[..., None]
        dy, ds = dy.masked_fill(padded, 0), ds.masked_fill_(padded, 0)
        return (scatter_rows(out), scatter_rows(ds @ key), scatter_columns(ds.transpose(2, 3) @ query),
                scatter_columns(p.transpose(2, 3) @ dy))


def _newton_schulz(x):
    """Five Newton-Schulz steps of a stack of matrices [count, short, long] in 32 bits."""
    a, b, c = COEFFICIENTS
    x = x / x.double().square().sum((1, 2), keepdim=True).sqrt().float().clamp(min=EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def _plain_newton_schulz(matrices):
    """The matrices in 32 bits after the iteration, those of one shape together."""
    together = {}
    for i, m in enumerate(matrices):
        together.setdefault(tuple(m.shape), []).append(i)
    results = [None] * len(matrices)
    for (rows, cols), members in together.items():
        x = torch.stack([matrices[i] for i in members]).float()
        x = _newton_schulz(x.transpose(1, 2)).transpose(1, 2) if rows > cols else _newton_schulz(x)
        for i, y in zip(members, x):
            results[i] = y
    return results


def _plain_orthogonalize(matrices):
    return [y.to(m.dtype) for m, y in zip(matrices, _plain_newton_schulz(matrices))]


def _plain_muon(state):
    lr, mu, decay = MUON["lr"], MUON["momentum"], MUON["weight_decay"]
    with torch.no_grad():
        updates = []
        for p, m in zip(state["params"], state["buffers"]):
            g = p.grad.float()
            m.mul_(mu).add_(g, alpha=1 - mu)
            updates.append((1 - mu) * g + mu * m)
        for p, y in zip(state["params"], _plain_newton_schulz(updates)):
            factor = lr * math.sqrt(max(1, p.shape[0] / p.shape[1]))
            p.copy_(p.float() * (1 - lr * decay) - factor * y)
    return tuple(state["params"]) + tuple(state["buffers"])


# ----------------------------------------------------------------------------- what a pass needs
def _pairs(case):
    """Query-key pairs that the mask leaves, per head."""
    total = 0
    for lq, lk in zip(_sizes(case["queries"]), _sizes(case["keys"])):
        if not case["causal"]:
            total += lq * lk
        else:  # query i sees keys 0 .. i + lk - lq
            first = max(0, lq - lk)
            count = lq - first
            low = first + lk - lq + 1
            total += count * (low + lk) // 2
    return total


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "attention":
        dim = case["head_dim"]
        rows = sum(_sizes(case["queries"])) * case["heads"] * dim
        columns = sum(_sizes(case["keys"])) * case["kv_heads"] * dim
        product = 2.0 * _pairs(case) * case["heads"] * dim
        if case["direction"] == "forward":
            return {"bytes": float(size * (2 * rows + 2 * columns)), "flops": 2 * product}
        # forward: q, k, v read, out written; backward: q, k, v, out, dy read, the gradients written
        return {"bytes": float(size * (5 * rows + 6 * columns)), "flops": 7 * product}
    shapes = _matrix_shapes(case)
    numel = sum(rows * cols for rows, cols in shapes)
    # The iteration lives in the short side's Gram matrix: one product makes it (half of it, by
    # symmetry), one applies the result, and 17 symmetric products of the short side lie between.
    flops = sum(3.0 * min(s) ** 2 * max(s) + 17.0 * min(s) ** 3 for s in shapes)
    if case["kind"] == "orthogonalize":
        return {"bytes": float(2 * size * numel), "flops": flops}
    return {"bytes": float((3 * size + 8) * numel), "flops": flops}


# ----------------------------------------------------------------------------- in 64 bits
def _exact_attention(case, state):
    q, k, v = (state[name].detach().double() for name in ("q", "k", "v"))
    group = case["heads"] // case["kv_heads"]
    train = case["direction"] == "train"
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for (qa, qb), (ka, kb) in zip(_records(_sizes(case["queries"])), _records(_sizes(case["keys"]))):
        allowed = torch.ones(qb - qa, kb - ka, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            allowed = allowed.tril((kb - ka) - (qb - qa))
        blocked = torch.zeros(allowed.shape, dtype=torch.float64, device=DEVICE).masked_fill_(~allowed, -math.inf)
        for h in range(case["heads"]):
            key, value = k[ka:kb, h // group], v[ka:kb, h // group]
            p = torch.softmax(q[qa:qb, h] @ key.T / case["head_dim"] ** 0.5 + blocked, -1).nan_to_num(0.0)
            out[qa:qb, h] = p @ value
            if train:
                upstream = state["dy"][qa:qb, h].double()
                dv[ka:kb, h // group] += p.T @ upstream
                dp = upstream @ value.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / case["head_dim"] ** 0.5
                dq[qa:qb, h] = ds @ key
                dk[ka:kb, h // group] += ds.T @ q[qa:qb, h]
    return (out, dq, dk, dv) if train else out


def _exact_orthogonal(matrix):
    a, b, c = COEFFICIENTS
    x = matrix.double()
    x = x / max(float(torch.linalg.matrix_norm(x)), EPS)
    tall = x.shape[0] > x.shape[1]
    for _ in range(STEPS):
        if tall:
            square = x.T @ x
            x = a * x + x @ (b * square + c * square @ square)
        else:
            square = x @ x.T
            x = a * x + (b * square + c * square @ square) @ x
    return x


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "attention":
            return _exact_attention(case, state)
        if case["kind"] == "orthogonalize":
            return [_exact_orthogonal(m) for m in state["matrices"]]
        params, buffers = [], []
        for p, m in zip(state["params"], state["buffers"]):
            g, old = p.grad.double(), m.double()
            new = MUON["momentum"] * old + (1 - MUON["momentum"]) * g
            direction = _exact_orthogonal(MUON["momentum"] * new + (1 - MUON["momentum"]) * g)
            factor = MUON["lr"] * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            params.append(p.double() * (1 - MUON["lr"] * MUON["weight_decay"]) - factor * direction)
            buffers.append(new)
    return tuple(params) + tuple(buffers)
