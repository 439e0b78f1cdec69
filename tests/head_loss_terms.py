"""Inputs and bounds of the streamed losses where exponentials or derivatives are held in two bf16 terms: a term that
is lost shows."""

import torch

from head_loss_reference import bounds, reference


COLUMNS = 16   # the others are zero, so that no product or sum of theirs rounds


def inputs(rows, width, offset, device):
    """float32 values that bf16 holds; logits around `offset` with a few large ones in a row (a row's gradient then is
    that of a few exponentials, whose roundings do not average). At 33 the units of 128 entries lie on both sides
    of 48 log 2, where their shifts step, and are brought to their row's."""
    g = torch.Generator().manual_seed(rows + width)
    hidden, head = torch.zeros(rows, width), torch.zeros(700, width)
    hidden[:, :15] = torch.randn(rows, 15, generator=g)
    head[:, :15] = torch.randn(700, 15, generator=g)
    hidden[:, 15], head[:, 15] = 1.0, offset
    labels = torch.randint(700, (rows,), generator=g)
    weights = torch.rand(rows, generator=g) + 0.1
    round_ = lambda t: t.bfloat16().float().to(device)  # noqa: E731
    return round_(hidden), round_(head), labels.to(device), weights.to(device)


def expected(hidden, head, labels, weights):
    """(loss, dh, dW, parts) of the first COLUMNS and the bounds of both gradients: those of float32 results, and 2^-16 of every exponential
    (of the derivative) beside: what two bf16 terms leave, each half a step of 2^-7 of what it rounds."""
    want = reference(hidden[:, :COLUMNS], head[:, :COLUMNS], labels[:, None], None, weights)
    h, w, c, _, q, mass, _, p, d = want[3]
    _, dh, dw = bounds(want[3], weights, torch.float32, torch.float32, torch.float32)
    dh = dh + 2.0 ** -16 * (torch.where(q > 0, 0.0, c.abs()[:, None] * mass[:, None] * p) @ w.abs())
    dw = dw + 2.0 ** -16 * (d.abs().T @ h.abs())
    return want, dh, dw
