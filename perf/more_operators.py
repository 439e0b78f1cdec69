"""The end of a decoder in training: the final layer norm, the head's cross-entropy walked in
pieces of the vocabulary, and distillation from a teacher's top logits.

`listed()` names the cases, `draw(rng)` makes further ones of the same ranges, `prepare(case,
seed)` builds what a training program has in hand, and `run(state)` is one pass: through the
framework's operators where `own` is true, through their plain form in elementary float32
operations otherwise. `exact` states the same in float64 through autograd, `work` what a pass
cannot do without.
"""

import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "causal-tuner_amd"))

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5
_LARGEST = 16384 * 2048 * 49152   # rows x width x vocabulary of the largest loss


def listed():
    return [
        # One supervised token, the smallest call: an answer of one token, scored and trained on.
        {"name": "loss-token", "kind": "loss", "rows": 1, "tokens": 1, "width": 2048, "vocab": 49152,
         "dtype": "bf16", "grads": "hidden"},
        # A short batch on an odd vocabulary, the head trained with it.
        {"name": "loss-short-batch", "kind": "loss", "rows": 257, "tokens": 257, "width": 1000, "vocab": 32003,
         "dtype": "bf16", "grads": "both"},
        # An adapter's training step: the answers' tokens among the prompts', a frozen head.
        {"name": "loss-scattered", "kind": "loss", "rows": 2665, "tokens": 4096, "width": 2048, "vocab": 49152,
         "dtype": "bf16", "grads": "hidden"},
        # The same with the head trained too.
        {"name": "loss-trained-head", "kind": "loss", "rows": 4001, "tokens": 4001, "width": 2048, "vocab": 49152,
         "dtype": "bf16", "grads": "both"},
        # A long batch, every token supervised, a frozen head: the largest.
        {"name": "loss-long-batch", "kind": "loss", "rows": 16384, "tokens": 16384, "width": 2048, "vocab": 49152,
         "dtype": "bf16", "grads": "hidden"},
        # Training in float32, sizes that fill no tile.
        {"name": "loss-float32", "kind": "loss", "rows": 500, "tokens": 611, "width": 1022, "vocab": 32001,
         "dtype": "f32", "grads": "both"},
        # A few tokens from a teacher's eight best.
        {"name": "distill-few-tokens", "kind": "distill", "rows": 16, "tokens": 16, "width": 2048, "vocab": 49152,
         "entries": 8, "temperature": 1.0, "ragged": False, "normalizer": False, "dtype": "bf16", "grads": "hidden"},
        # A batch of stored teacher answers, softened, a frozen head.
        {"name": "distill-batch", "kind": "distill", "rows": 8192, "tokens": 8192, "width": 2048, "vocab": 49152,
         "entries": 64, "temperature": 2.0, "ragged": False, "normalizer": False, "dtype": "bf16",
         "grads": "hidden"},
        # Nucleus-cut lists of different lengths with the teacher's own normalizer, the head trained.
        {"name": "distill-ragged", "kind": "distill", "rows": 1500, "tokens": 2001, "width": 1024, "vocab": 50257,
         "entries": 20, "temperature": 1.0, "ragged": True, "normalizer": True, "dtype": "bf16", "grads": "both"},
        # One token answered: forward alone, where latency counts.
        {"name": "norm-token", "kind": "norm", "rows": 1, "width": 2048, "dtype": "bf16", "weights": "bf16",
         "bias": True, "grads": False},
        # A long batch of a wide model, forward and backward with the weight's gradient.
        {"name": "norm-batch", "kind": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "weights": "bf16",
         "bias": True, "grads": True},
        # float32 rows that fill no vector, no bias.
        {"name": "norm-ragged", "kind": "norm", "rows": 3001, "width": 1023, "dtype": "f32", "weights": "f32",
         "bias": False, "grads": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "distill", "norm"])
    if kind == "norm":
        width = _spread(rng, 16, 16384)
        rows = min(_spread(rng, 1, 65536), 16384 * 4096 // width)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        return {"kind": kind, "rows": rows, "width": width, "dtype": dtype,
                "weights": rng.choice(["bf16", "f32"]) if dtype == "bf16" else "f32", "bias": rng.random() < 0.7,
                "grads": rng.random() < 0.8}
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    width = _spread(rng, 64, 4096)
    if dtype == "bf16" and rng.random() < 0.8:
        width = width // 8 * 8
    vocab = _spread(rng, 300, 131072)
    rows = _spread(rng, 1, 8192 if dtype == "bf16" else 512)
    grads = rng.choice(["hidden", "both"])
    rows = max(1, min(rows, _LARGEST // (width * vocab) * 2 // (3 if grads == "both" else 2)))
    case = {"kind": kind, "rows": rows, "tokens": rows + (rng.randrange(rows + 1) if rng.random() < 0.5 else 0),
            "width": width, "vocab": vocab, "dtype": dtype, "grads": grads}
    if kind == "distill":
        case.update(entries=_spread(rng, 1, 128), temperature=rng.choice([0.5, 1.0, 2.0, 4.0]),
                    ragged=rng.random() < 0.5, normalizer=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, generator, scale=1.0):
    return torch.randn(shape, generator=generator, device="cuda") * scale


def _chunks(rows, vocab):
    step = max(1, min(rows, (1 << 28) // vocab))
    return [slice(a, min(a + step, rows)) for a in range(0, rows, step)]


def _loss_state(case, seed):
    """Hidden states with a common direction, as a final norm leaves them; a head whose logits
    spread over a few units; labels drawn from a sharper model of the same states, so that most
    tokens are likely and some are not."""
    g = _generator(seed)
    dtype, tokens, rows = _DTYPES[case["dtype"]], case["tokens"], case["rows"]
    width, vocab = case["width"], case["vocab"]
    hidden = (_normal((tokens, width), g) + _normal((width,), g, 0.3)).to(dtype)
    head = _normal((vocab, width), g, 2.5 / math.sqrt(width)).to(dtype)
    where = None
    if rows < tokens:
        where = torch.randperm(tokens, generator=g, device="cuda")[:rows].sort().values
    weights = torch.zeros(tokens, device="cuda")
    each = (0.5 + torch.rand(rows, generator=g, device="cuda")) / rows
    weights[slice(0, rows) if where is None else where] = each
    hidden.requires_grad_(True)
    head.requires_grad_(case["grads"] == "both")
    state = {"kind": case["kind"], "hidden": hidden, "head": head, "weights": weights,
             "rows": slice(0, rows) if where is None else where, "dtype": dtype}
    wide = hidden.detach().to(torch.bfloat16)
    matrix = head.detach().to(torch.bfloat16).T
    if case["kind"] == "loss":
        targets = torch.empty(tokens, dtype=torch.int64, device="cuda")
        for part in _chunks(tokens, vocab):
            logits = 1.5 * (wide[part] @ matrix).float()
            noise = torch.rand(logits.shape, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
            targets[part] = (logits - (-noise.log()).log()).argmax(-1)
        state["targets"] = targets
        return state
    entries = min(case["entries"], vocab)
    temperature = case["temperature"]
    indices = torch.empty((tokens, entries), dtype=torch.int64, device="cuda")
    values = torch.empty((tokens, entries), device="cuda")
    normalizer = torch.empty(tokens, device="cuda")
    for part in _chunks(tokens, vocab):
        teacher = wide[part].float() + _normal(wide[part].shape, g, 0.4)
        logits = 1.2 * (teacher.to(torch.bfloat16) @ matrix).float()
        values[part], indices[part] = logits.topk(entries, -1)
        normalizer[part] = torch.logsumexp(logits / temperature, -1)
    if case["ragged"]:
        kept = torch.randint(0, entries + 1, (tokens, 1), generator=g, device="cuda")
        gone = torch.arange(entries, device="cuda") >= kept
        indices = indices.masked_fill(gone, -1)
        values = values.masked_fill(gone, -math.inf)
    state.update(indices=indices, values=values, temperature=temperature,
                 normalizer=normalizer if case["normalizer"] else None)
    return state


def _norm_state(case, seed):
    g = _generator(seed)
    rows, width = case["rows"], case["width"]
    dtype, kept = _DTYPES[case["dtype"]], _DTYPES[case["weights"]]
    # a residual stream: channels of different size, rows with means of their own
    scale = torch.exp(_normal((width,), g, 0.5))
    x = (_normal((rows, width), g) * scale + _normal((rows, 1), g, 0.7)).to(dtype)
    weight = (1 + _normal((width,), g, 0.2)).to(kept)
    bias = _normal((width,), g, 0.1).to(kept) if case["bias"] else None
    grad = _normal((rows, width), g).to(dtype) if case["grads"] else None
    if case["grads"]:
        for leaf in (x, weight, bias):
            if leaf is not None:
                leaf.requires_grad_(True)
    return {"kind": "norm", "x": x, "weight": weight, "bias": bias, "grad": grad}


def prepare(case, seed):
    return _norm_state(case, seed) if case["kind"] == "norm" else _loss_state(case, seed)


# ------------------------------------------------------------------------------ one pass
def run(state):
    if state["kind"] == "norm":
        return _run_norm(state)
    return _run_loss(state)


def _run_norm(state):
    x, weight, bias, grad = state["x"], state["weight"], state["bias"], state["grad"]
    leaves = [t for t in (x, weight, bias) if t is not None]
    if own:
        from causal_tuner.modeling.norm import layer_norm
        y = layer_norm(x, weight, bias, _EPS)
        if grad is None:
            return {"y": y}
        return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, grad)}
    with torch.no_grad():
        wide = x.float()
        centred = wide - wide.mean(-1, keepdim=True)
        rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
        n = centred * rstd
        y = n * weight.float()
        if bias is not None:
            y = y + bias.float()
        y = y.to(x.dtype)
        if grad is None:
            return {"y": y}
        dy = grad.float()
        g = dy * weight.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
        grads = [dx.to(x.dtype), (dy * n).sum(0).to(weight.dtype)]
        if bias is not None:
            grads.append(dy.sum(0).to(bias.dtype))
        return {"y": y, "grads": grads}


def _leaves(state):
    return [t for t in (state["hidden"], state["head"]) if t.requires_grad]


def _run_loss(state):
    if own:
        from causal_tuner.kernels.loss import distillation_loss, projection_loss
        common = {"compute_dtype": state["dtype"], "rows": state["rows"]}
        if state["kind"] == "loss":
            loss = projection_loss(state["hidden"], state["head"], state["targets"], state["weights"],
                                   implementation="streamed", **common)
        else:
            loss = distillation_loss(state["hidden"], state["head"], state["indices"], state["values"],
                                     state["weights"], temperature=state["temperature"],
                                     log_normalizer=state["normalizer"], **common)
        return {"loss": loss.detach(), "grads": torch.autograd.grad(loss, _leaves(state))}
    with torch.no_grad():
        return _plain_loss(state)


def _plain_loss(state):
    """Every logit of the supervised rows at once, in float32."""
    hidden, head, rows = state["hidden"], state["head"], state["rows"]
    h, matrix, weights = hidden[rows].float(), head.float(), state["weights"][rows]
    if state["kind"] == "loss":
        temperature, index = 1.0, state["targets"][rows][:, None]
        q = torch.ones(index.shape, device=h.device)
        entropy = torch.zeros(len(h), device=h.device)
    else:
        temperature, index = state["temperature"], state["indices"][rows]
        given = index >= 0
        teacher = torch.where(given, state["values"][rows] / temperature, torch.tensor(-math.inf, device=h.device))
        if state["normalizer"] is not None:
            log_q = teacher - state["normalizer"][rows][:, None]
        else:
            top = teacher.amax(-1, keepdim=True).clamp_min(-1e30)
            log_q = teacher - top - (teacher - top).exp().sum(-1, keepdim=True).log()
        q = torch.where(given, log_q.exp(), torch.zeros_like(log_q))
        entropy = torch.where(given, q * log_q, torch.zeros_like(q)).sum(-1)
        index = index.clamp_min(0)
    logits = (h @ matrix.T).div_(temperature)
    top = logits.amax(-1, keepdim=True)
    chosen = logits.gather(1, index) - top
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    mass = q.sum(-1)
    loss = (weights * (entropy - (q * chosen).sum(-1) + mass * total[:, 0].log())).sum()
    d = p.mul_(mass[:, None] / total).scatter_add_(1, index, -q).mul_((weights / temperature)[:, None])
    grads = [torch.zeros_like(hidden)]
    grads[0][rows] = (d @ matrix).to(hidden.dtype)
    if head.requires_grad:
        grads.append((d.T @ h).to(head.dtype))
    return {"loss": loss, "grads": grads}


# ------------------------------------------------------------------------------ what it takes
def work(case):
    rows, width = case["rows"], case["width"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        kept = 2 if case["weights"] == "bf16" else 4
        vectors = width * kept * (2 if case["bias"] else 1)
        if not case["grads"]:
            return {"bytes": 2 * rows * width * size + vectors, "flops": 8 * rows * width}
        # the forward reads x and writes y, the backward reads x and dy and writes dx
        return {"bytes": 5 * rows * width * size + 3 * vectors, "flops": 22 * rows * width}
    vocab, both = case["vocab"], case["grads"] == "both"
    nbytes = size * (2 * rows * width + vocab * width * (2 if both else 1)) + rows * 12
    if case["kind"] == "distill":
        nbytes += rows * case["entries"] * 12
    # the logits, the hidden states' gradient and the head's
    return {"bytes": nbytes, "flops": 2 * rows * width * vocab * (3 if both else 2)}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(state)
    hidden = state["hidden"].detach().double().requires_grad_(True)
    head = state["head"].detach().double().requires_grad_(state["head"].requires_grad)
    leaves = [t for t in (hidden, head) if t.requires_grad]
    weights = state["weights"].double()
    rows = torch.arange(len(hidden), device="cuda")[state["rows"]]
    total, grads = 0.0, [torch.zeros_like(t) for t in leaves]
    for part in _chunks(len(rows), case["vocab"]):
        at = rows[part]
        scores = hidden[at] @ head.T
        if case["kind"] == "loss":
            terms = -torch.log_softmax(scores, -1)[torch.arange(len(at)), state["targets"][at]]
        else:
            terms = _exact_divergence(state, scores, at)
        loss = (terms * weights[at]).sum()
        total = total + loss.detach()
        for sum_, grad in zip(grads, torch.autograd.grad(loss, leaves)):
            sum_ += grad
    return {"loss": total, "grads": grads}


def _exact_divergence(state, scores, at):
    """sum over the teacher's entries of q (log q - log p), row by row."""
    temperature = state["temperature"]
    log_p = torch.log_softmax(scores / temperature, -1)
    index, values = state["indices"][at], state["values"][at].double() / temperature
    there = index >= 0
    if state["normalizer"] is not None:
        log_q = values - state["normalizer"][at].double()[:, None]
    else:
        log_q = values - torch.logsumexp(values.masked_fill(~there, -math.inf), -1, keepdim=True)
    log_q = log_q.masked_fill(~there, 0.0)
    q = log_q.exp().masked_fill(~there, 0.0)
    return (q * (log_q - log_p.gather(1, index.masked_fill(~there, 0)))).sum(-1)


def _exact_norm(state):
    leaves = [t.detach().double().requires_grad_(t.requires_grad)
              for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    x, weight = leaves[0], leaves[1]
    spread, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = (x - mean) / (spread + _EPS).sqrt() * weight
    if state["bias"] is not None:
        y = y + leaves[2]
    if state["grad"] is None:
        return {"y": y}
    return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, state["grad"].double())}
