"""The head's loss in float64 from its definition, and how far a result may be from it, counted from
the roundings of the kernels (see `bounds`)."""

import math

import torch


def targets(indices, values, temperature, normalizer, vocab):
    """Dense q [rows, vocab] in float64; `values` None: hard labels [rows, 1]."""
    there = (indices >= 0) & (indices < vocab)
    q = torch.zeros(len(indices), vocab, dtype=torch.float64, device=indices.device)
    if values is None:
        return q.scatter_add_(1, indices.clamp(0, vocab - 1), there.double())
    logits = (values.double() / temperature).masked_fill(~there, -math.inf)
    if normalizer is None:
        top = torch.logsumexp(logits, -1, keepdim=True)
        log_q = logits - torch.where(top == -math.inf, torch.zeros_like(top), top)
    else:
        log_q = logits - normalizer.double()[:, None]
    return q.scatter_add_(1, indices.clamp(0, vocab - 1), log_q.exp())


def reference(hidden, head, indices, values, weights, temperature=1.0, normalizer=None, upstream=1.0):
    """(loss, dh, dW, parts) of rows [N, d], all of them in the loss."""
    h, w, c = hidden.detach().double(), head.detach().double(), weights.double() * upstream / temperature
    logits = h @ w.T / temperature
    q = targets(indices, values, temperature, normalizer, len(w))
    # a hard label outside the vocabulary leaves log Z
    mass = torch.ones(len(h), dtype=torch.float64, device=h.device) if values is None else q.sum(-1)
    lse = torch.logsumexp(logits, -1)
    entropy = torch.where(q > 0, q * q.clamp_min(1e-300).log(), 0).sum(-1)
    row_loss = entropy + mass * lse - torch.where(q > 0, q * logits, 0).sum(-1)
    loss = (weights.double() * torch.where(mass > 0, row_loss, 0)).sum()
    # relative to the row's maximum: lse itself is rounded to 2^-53 of its size, which is more than
    # 1 - p of a confident row
    e = (logits - logits.amax(-1, keepdim=True)).exp()
    p = e / e.sum(-1, keepdim=True)
    d = mass[:, None] * p - q
    if values is None:   # 1 - p of the label: the others' share
        others = e.scatter(1, indices.clamp(0, len(w) - 1), 0.0).sum(-1) / e.sum(-1)
        d = torch.where(q > 0, -others[:, None], d)
    d = c[:, None] * d
    return loss, d @ w, d.T @ h, (h, w, c, logits, q, mass, lse, p, d)


def bounds(parts, weights, dtype, out_hidden, out_head, temperature=1.0):
    """Elementwise bounds of loss, dh and dW.

    A logit is a float32 chain of `width` products (2^-24 each, of the sum of magnitudes), times
    log2(e) / T rounded twice; the exponent's rounding, the exponential's own error and the sums' add
    up to 2^-17 of a probability (exponents reach 128 against a shift of 48 + 96 n: half an ulp there
    is 2^-18 times log 2). For bf16 the exponentials, or the derivative in the head's product, are rounded
    once more (half a step, 2^-8), but not the targets' terms of dh. Sums over the vocabulary or
    the rows add their length times 2^-24; the result is rounded to its own type."""
    h, w, c, logits, q, mass, lse, p, d = parts
    rows, width, vocab = len(h), h.shape[1], len(w)
    unit = 2.0 ** -24
    near = (width + 4) * unit * (h.abs() @ w.abs().T) / temperature + 4 * unit * logits.abs()
    far = near.amax(-1)
    off = 2 * far + 2.0 ** -17 + vocab * unit                        # relative, of every probability
    narrow = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    size = {torch.bfloat16: 2.0 ** -8, torch.float32: unit}
    loss = (weights.double() * mass * (2 * far + vocab * unit + 2.0 ** -20
                                       + 8 * unit * (lse.abs() + logits.abs().amax(-1)))).sum()
    spread = c.abs()[:, None] * mass[:, None] * p
    target = q > 0
    e = spread * (off[:, None] + torch.where(target, 0.0, narrow) + vocab * unit) + d.abs() * (vocab + 8) * unit
    e = e + torch.where(target, c.abs()[:, None] * q * 2.0 ** -20, 0.0)
    dh = e @ w.abs()
    g = spread * off[:, None] + d.abs() * (narrow + (rows + 8) * unit) + c.abs()[:, None] * q * 2.0 ** -20
    dw = g.T @ h.abs()
    exact_h, exact_w = d @ w, d.T @ h
    tiny = 1e-30
    return (loss + unit * 4 * loss, dh + size[out_hidden] * (exact_h.abs() + dh) + tiny,
            dw + size[out_head] * (exact_w.abs() + dw) + tiny)


def check(name, got, want, bound):
    error = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (error / bound).max().item() if error.numel() else 0.0
    assert worst <= 1, f"{name}: {worst:.3g} times its bound"
