"""Projection + weighted cross-entropy without ever holding the sequence's logits, and
distillation from a teacher's top logits in the same way (`distillation_loss`).

Interface of the reference's kernels/loss.py (`active_rows` 6-16, `row_count` 19-20,
`projection_loss` 23-66) and of its host autograd function `ProjectionLoss`
(kernels/reference.py:30-73). Device inputs take `loss_cuda.FusedProjectionLoss`; host
inputs take `ProjectionLoss` below. Both visit the supervised rows in tiles of at most
`token_budget` rows.
"""

import torch
import torch.nn.functional as F


def active_rows(weights, device=None):
    """The rows with weight > 0, chosen where the weights live. No supervised rows, or all
    of them, give a slice; host weights whose supervised rows form one interval give that
    slice (so the loss reads views and gathers nothing); otherwise the row indices, moved
    to `device` when given."""
    supervised = weights.flatten() > 0
    total = supervised.numel()
    count = int(supervised.sum())
    if count in (0, total):
        return slice(0, count)
    if weights.device.type == "cpu":
        first = int(supervised.to(torch.uint8).argmax())
        last = total - 1 - int(supervised.flip(0).to(torch.uint8).argmax())
        if last - first + 1 == count:
            return slice(first, last + 1)
    indices = supervised.nonzero().flatten()
    return indices if device is None else indices.to(device)


def row_count(rows):
    if isinstance(rows, slice):
        return rows.stop - rows.start
    return len(rows)


def _check_backend(implementation, cut_chunk_size, head):
    """The reference's backend options: 'fused' is the path here; 'cut' (the
    cut-cross-entropy package, not carried by this framework) is refused as it refuses it."""
    if implementation == "cut":
        if head.requires_grad:
            raise ValueError("cut cannot guarantee FP32 head-gradient accumulation; use fused")
        raise RuntimeError("The cut backend requires cut-cross-entropy")
    if implementation not in ("fused", "streamed"):
        raise ValueError("Unsupported projection-loss backend")
    if cut_chunk_size:
        raise ValueError("cut_chunk_size applies only to the cut backend")


def projection_loss(hidden, head, targets, weights, *, token_budget=128, compute_dtype=torch.bfloat16,
                    implementation="fused", cut_chunk_size=0, reuse_hidden=False, rows=None):
    """sum_i weights[i] * CE(hidden[i] head^T, targets[i]) over the supervised rows, with at
    most `token_budget` rows of logits at a time. `reuse_hidden` lets the gradient of
    `hidden` take over its storage (an exclusive contiguous non-leaf tensor). `rows` is a
    precomputed `active_rows` selection.

    `implementation="streamed"` takes all rows at once and walks the vocabulary in pieces instead
    (`head_loss_cuda`): no logits are held, so `token_budget` plays no part; the statistics and
    the loss come from unrounded float32 logits, and every gradient is rounded once, after the
    upstream scale. bf16 and float32; `reuse_hidden` belongs to the fused path, and weights that ask for
    a gradient are refused. With `rows` given it can be captured into a graph. `rows` are numbers
    counted from 0, in any order: one given twice counts twice, one that names no row has no loss."""
    if token_budget <= 0:
        raise ValueError("loss_token_budget must be positive")
    selection = active_rows(weights, hidden.device) if rows is None else rows
    if hidden.is_cuda and head.requires_grad and head.dtype == torch.float32:
        # The logits GEMM is the BLAS library's: its bf16 reductions stay in fp32.
        torch.backends.cuda.matmul.allow_bf16_reduced_precision_reduction = False
    _check_backend(implementation, cut_chunk_size, head)
    if implementation == "streamed":
        if reuse_hidden:
            raise ValueError("reuse_hidden applies only to the fused backend")
        if targets.is_floating_point():
            raise ValueError("targets are whole numbers")
        _check_rows(hidden, head, weights, {"targets": targets})
    if not hidden.is_cuda:
        if implementation == "streamed":
            selection, weights = _counted_rows(_named_rows(selection, weights.numel()), weights)
        return ProjectionLoss.apply(hidden, head, targets, weights, token_budget, compute_dtype, selection)
    if not torch.is_grad_enabled():
        hidden, head = hidden.detach(), head.detach()
    if implementation == "streamed":
        from .head_loss_cuda import streamed_loss
        return streamed_loss(hidden, head, weights, selection, compute_dtype, targets.reshape(-1, 1))
    if reuse_hidden and hidden.requires_grad:
        shared = hidden.is_leaf or hidden._base is not None or not hidden.is_contiguous()
        if shared:
            raise ValueError("Hidden reuse requires an exclusive contiguous non-leaf tensor")
    from .loss_cuda import FusedProjectionLoss
    total, _ = FusedProjectionLoss.apply(hidden, head, targets, weights, token_budget, compute_dtype,
                                         reuse_hidden, selection)
    return total


def _named_rows(selection, tokens):
    """Of row numbers on the host those that name a row, as the device's kernels take them: one outside [0, tokens)
    has no loss. A mask or a list is taken as its numbers."""
    if isinstance(selection, slice):
        return selection
    selection = torch.as_tensor(selection)
    if selection.numel() == 0:
        return slice(0, 0)
    if selection.dtype == torch.bool:
        return selection.nonzero().flatten()
    return selection[(selection >= 0) & (selection < tokens)]


def _counted_rows(selection, weights):
    """Row numbers without repeats, the weights of repeated ones times their count."""
    if isinstance(selection, slice):
        return selection, weights
    rows, times = selection.unique(return_counts=True)
    if len(rows) == len(selection):
        return selection, weights
    weights = weights.flatten().clone()
    weights[rows] *= times
    return rows, weights


def _check_rows(hidden, head, weights, tables):
    """One row of every table and one weight per row of hidden, all on its device."""
    if hidden.dim() < 1 or head.dim() != 2 or hidden.shape[-1] != head.shape[1] or head.numel() == 0:
        raise ValueError(f"hidden {tuple(hidden.shape)} and head {tuple(head.shape)} do not give logits")
    tokens = hidden.numel() // hidden.shape[-1]
    if weights.numel() != tokens:
        raise ValueError(f"{weights.numel()} weights for {tokens} rows of hidden")
    for name, table in tables.items():
        if table.numel() != tokens * (table.shape[-1] if name in ("indices", "values") else 1):
            raise ValueError(f"{name} {tuple(table.shape)} for {tokens} rows of hidden")
    if weights.requires_grad and torch.is_grad_enabled():
        raise ValueError("weights get no gradient: detach them")
    for name, table in {"head": head, **tables}.items():
        if table.device != hidden.device:
            raise ValueError(f"{name} is on {table.device}, hidden on {hidden.device}")


def distillation_loss(hidden, head, indices, values, weights, *, temperature=1.0, log_normalizer=None,
                      compute_dtype=torch.bfloat16, rows=None):
    """Distillation from a teacher's top logits: over the supervised rows,

        sum_i weights[i] * sum_k q_ik (log q_ik - log p_i[indices[i, k]]),
        p_i = softmax(hidden[i] head^T / temperature) over the whole vocabulary,
        q_i = softmax(values[i] / temperature) over the row's entries, or, with `log_normalizer`
              (the teacher's own log sum exp of its logits / temperature, one per row),
              exp(values[i] / temperature - log_normalizer[i]), whose sum may be below one.

    `indices` and `values` are [..., K], K up to 1024, one row per row of hidden. Lists may differ in length:
    an index outside [0, vocab) (-1, say) is no entry, whatever its value; a value of -inf is an
    entry without mass; an index given twice counts once, with the sum of both probabilities; a row
    without entries has no loss and no gradient. The factor temperature^2 that keeps the gradient's size,
    or a share beside another loss, belongs into `weights`. The vocabulary is walked in pieces
    as `projection_loss(implementation="streamed")` does, on the same kernels; gradients reach
    hidden and head, not the teacher or the weights, which are refused where they ask for one. `rows`
    as in `projection_loss`."""
    if indices.dim() < 1 or indices.shape != values.shape:
        raise ValueError(f"indices {tuple(indices.shape)} and values {tuple(values.shape)} differ")
    if not 1 <= indices.shape[-1] <= 1024:
        raise ValueError(f"{indices.shape[-1]} entries per row: 1 to 1024 are taken")
    if indices.is_floating_point() or not values.is_floating_point():
        raise ValueError("indices are whole numbers, values floating")
    temperature = float(temperature)
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
        raise ValueError(f"temperature {temperature} is not a positive number between 2^-60 and 2^60")
    tables = {"indices": indices, "values": values}
    if log_normalizer is not None:
        tables["log_normalizer"] = log_normalizer
    _check_rows(hidden, head, weights, tables)
    if any(t is not None and t.requires_grad for t in (values, log_normalizer)):
        raise ValueError("the teacher's values get no gradient: detach them")
    selection = active_rows(weights, hidden.device) if rows is None else rows
    entries = indices.shape[-1]
    indices, values = indices.reshape(-1, entries), values.reshape(-1, entries)
    log_normalizer = None if log_normalizer is None else log_normalizer.flatten()
    if not hidden.is_cuda:
        return _host_distillation(hidden, head, indices, values, weights, temperature, log_normalizer, compute_dtype,
                                  selection)
    if not torch.is_grad_enabled():
        hidden, head = hidden.detach(), head.detach()
    from .head_loss_cuda import streamed_loss
    return streamed_loss(hidden, head, weights, selection, compute_dtype, indices, values, log_normalizer, temperature)


def _host_distillation(hidden, head, indices, values, weights, temperature, log_normalizer, compute_dtype, selection):
    """The same in torch operations, float32 (float64 for its tensors) from the logits on."""
    selection = _named_rows(selection, len(indices))
    h = hidden.reshape(-1, hidden.shape[-1])[selection].to(compute_dtype)
    wide = torch.promote_types(compute_dtype, torch.float32)
    log_p = torch.log_softmax(F.linear(h, head.to(compute_dtype)).to(wide) / temperature, -1)
    index, scale = indices[selection], weights.flatten()[selection].to(wide)
    teacher = (values[selection].to(wide) / temperature).masked_fill((index < 0) | (index >= len(head)), -float("inf"))
    if log_normalizer is None:
        # a row without any mass has no entries
        log_q = teacher - torch.logsumexp(teacher, -1, keepdim=True).clamp_min(torch.finfo(wide).min)
    else:
        log_q = teacher - log_normalizer[selection].to(wide)[:, None]
    q = torch.zeros_like(log_p).scatter_add_(1, index.clamp(0, len(head) - 1), log_q.exp())
    return (scale[:, None] * torch.where(q != 0, q * (torch.where(q != 0, q, 1).log() - log_p), 0)).sum()


def _host_tiles(selection, tile):
    """(row selector, size) of each tile of the supervised rows."""
    count = row_count(selection)
    for offset in range(0, count, tile):
        size = min(tile, count - offset)
        if isinstance(selection, slice):
            yield slice(selection.start + offset, selection.start + offset + size), size
        else:
            yield selection[offset:offset + size], size


class ProjectionLoss(torch.autograd.Function):
    """Host route. Per tile the logits are formed in the compute dtype and widened to fp32
    for the CE; the backward forms them again (nothing but the inputs is saved), rounds the
    weighted softmax derivative (scaled by the upstream value) to the compute dtype, and
    accumulates d head in fp32 for an fp32 head."""

    @staticmethod
    def forward(ctx, hidden, head, targets, weights, tile, compute_dtype, active):
        ctx.tile, ctx.compute_dtype = tile, compute_dtype
        ctx.interval = active if isinstance(active, slice) else None
        ctx.save_for_backward(hidden, head, targets, weights, None if ctx.interval is not None else active)
        h, labels, scale = hidden.reshape(-1, hidden.shape[-1]), targets.flatten(), weights.flatten()
        matrix = head.to(compute_dtype)
        total = torch.zeros((), device=hidden.device, dtype=torch.float32)
        for where, _ in _host_tiles(active, tile):
            logits = F.linear(h[where].to(compute_dtype), matrix).float()
            total += (F.cross_entropy(logits, labels[where], reduction="none") * scale[where]).sum()
        return total

    @staticmethod
    def backward(ctx, upstream):
        hidden, head, targets, weights, indices = ctx.saved_tensors
        active = ctx.interval if ctx.interval is not None else indices
        dtype = ctx.compute_dtype
        h, labels, scale = hidden.reshape(-1, hidden.shape[-1]), targets.flatten(), weights.flatten()
        matrix = head.to(dtype)
        d_hidden = torch.zeros_like(h) if ctx.needs_input_grad[0] else None
        d_head = torch.zeros_like(head) if ctx.needs_input_grad[1] else None
        for where, size in _host_tiles(active, ctx.tile):
            x = h[where].to(dtype)
            probabilities = F.linear(x, matrix).float().softmax(dim=-1)
            probabilities[torch.arange(size), labels[where]] -= 1
            derivative = (probabilities * (scale[where] * upstream)[:, None]).to(dtype)
            if d_hidden is not None:
                d_hidden[where] = (derivative @ matrix).to(d_hidden.dtype)
            if d_head is None:
                continue
            if head.dtype == torch.float32:
                d_head.addmm_(derivative.float().T, x.float())   # fp32 product, fp32 sums
            else:
                d_head += (derivative.T @ x).to(d_head.dtype)
        result = None if d_hidden is None else d_hidden.reshape_as(hidden)
        return result, d_head, None, None, None, None, None
