"""The head's loss over a vocabulary walked in pieces on gfx950 (ct_head_loss_forward,
ct_head_loss_backward): behind `loss.projection_loss(implementation="streamed")` (hard labels) and
`loss.distillation_loss` (a teacher's top logits), which state what is computed.

No logits are held. The forward makes a running softmax over the pieces and, in the same sweep,
the float32 sums behind the hidden rows' gradient; what it keeps for the backward are those sums,
two numbers per row and the targets. The backward scales the sums by the upstream value, adds the
targets' own terms and rounds once; the head's gradient forms the logits again, piece by piece. A backward may
be repeated. Results do not depend on timing: repeated calls are bit-identical.
"""

import torch

from . import _native
from .loss import row_count


def _rows_of(selection, tokens, device):
    """(first row, row indices or None, count) of a selection."""
    if isinstance(selection, slice):
        first, stop, _ = selection.indices(tokens)
        if selection.step not in (None, 1):
            raise ValueError("rows: a slice of consecutive rows")
        return first, None, max(stop - first, 0)
    if selection.dtype == torch.bool or selection.is_floating_point() or selection.dim() != 1:
        raise ValueError("rows: a slice or a vector of row numbers")
    return 0, selection.to(device, torch.int64).contiguous(), row_count(selection)


def _aligned_head(head):
    """`head` with unit-stride rows that start at 16-byte boundaries, bf16 widths a multiple of 8:
    itself, or a copy padded with zeros."""
    if head.dtype != torch.bfloat16:
        return head if head.stride(1) == 1 and head.stride(0) >= head.shape[1] else head.contiguous()
    pad = -head.shape[1] % 8
    if pad:
        return torch.nn.functional.pad(head, (0, pad))
    if head.stride(1) != 1 or head.stride(0) % 8 or head.stride(0) < head.shape[1] or head.data_ptr() % 16:
        return head.clone(memory_format=torch.contiguous_format)
    return head


def _plain_rows(hidden):
    h = hidden.reshape(-1, hidden.shape[-1])
    return h if h.stride(1) == 1 and h.stride(0) >= h.shape[1] else h.contiguous()


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


class _Call:
    """The C call's operands, and the tensors they point into."""

    def __init__(self, hidden, matrix, tables, first, rows, count, temperature):
        indices, values, normalizer, weights = tables
        self.held = (hidden, matrix, tables, rows)
        size = hidden.element_size()
        shift = lambda t, pitch: None if t is None else t.data_ptr() + first * pitch * t.element_size()  # noqa: E731
        entries = indices.shape[1]
        self.c = _native.HeadLoss(
            hidden=hidden.data_ptr() + first * hidden.stride(0) * size, head=matrix.data_ptr(), rows=_native.ptr(rows),
            indices=shift(indices, entries), values=shift(values, entries), log_normalizer=shift(normalizer, 1),
            weights=shift(weights, 1), ld_hidden=max(hidden.stride(0), hidden.shape[1]), ld_head=matrix.stride(0),
            ld_indices=entries, ld_values=entries, tokens=len(hidden) - first, hidden_width=hidden.shape[1], count=count,
            width=matrix.shape[1], vocab=len(matrix), entries=entries, dtype=_native.dtype_code(matrix.dtype),
            temperature=temperature)
        self.sizes = (count, matrix.shape[1], len(matrix), entries, self.c.dtype)


class StreamedHeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, head, tables, selection, compute_dtype, temperature):
        need_hidden, need_head = ctx.needs_input_grad[:2]
        h, matrix = _plain_rows(hidden.to(compute_dtype)), _aligned_head(head.to(compute_dtype))
        first, rows, count = _rows_of(selection, len(h), h.device)
        call = _Call(h, matrix, tables, first, rows, count, temperature)
        lib = _native.library()
        loss = torch.empty((), dtype=torch.float32, device=h.device)
        kept = _workspace(lib.ct_head_loss_kept(*call.sizes, int(need_hidden)), h.device)
        scratch = _workspace(lib.ct_head_loss_workspace(*call.sizes, int(need_hidden)), h.device)
        with _native.device_of(h):
            status = lib.ct_head_loss_forward(call.c, loss.data_ptr(), int(need_hidden), kept.data_ptr(), kept.numel(),
                                              scratch.data_ptr(), scratch.numel(), _native.stream_of(h))
        _native.check(status, "ct_head_loss_forward")
        indices, values, normalizer, weights = tables
        ctx.save_for_backward(h if need_head else None, matrix, kept, indices, values, normalizer, weights, rows)
        ctx.call = (first, count, temperature, need_hidden, hidden.shape, hidden.dtype, head.shape, head.dtype)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        h, matrix, kept, indices, values, normalizer, weights, rows = ctx.saved_tensors
        first, count, temperature, kept_sums, hidden_shape, hidden_dtype, head_shape, head_dtype = ctx.call
        _native.refuse_tangents("projection_loss", upstream)
        device, width = matrix.device, head_shape[1]
        tokens = hidden_shape[:-1].numel()
        d_hidden = d_head = hidden_out = head_out = None
        if ctx.needs_input_grad[0]:
            dtype = hidden_dtype if hidden_dtype == torch.bfloat16 else torch.float32
            fresh = torch.empty if rows is None and count == tokens else torch.zeros
            d_hidden = fresh((tokens, width), dtype=dtype, device=device)
            hidden_out = d_hidden[first:]
        if ctx.needs_input_grad[1]:
            narrow = head_dtype == torch.bfloat16 and matrix.dtype == torch.bfloat16
            fresh = torch.empty if count else torch.zeros
            d_head = head_out = fresh(head_shape, dtype=torch.bfloat16 if narrow else torch.float32, device=device)
        if count:
            # without the head's gradient the hidden rows are not read: any rows stand for them
            rows_in = h if h is not None else d_hidden
            call = _Call(rows_in, matrix, (indices, values, normalizer, weights), first, rows, count, temperature)
            upstream = upstream.to(torch.float32)
            lib = _native.library()
            scratch = _workspace(lib.ct_head_loss_workspace(*call.sizes, 2) if d_head is not None else 0, device)
            code = lambda t: _native.CT_F32 if t is None else _native.dtype_code(t.dtype)  # noqa: E731
            with _native.device_of(matrix):
                status = lib.ct_head_loss_backward(
                    call.c, upstream.data_ptr(), kept.data_ptr(), int(kept_sums), kept.numel(), _native.ptr(hidden_out),
                    width, width, code(d_hidden), _native.ptr(head_out), width, width, code(d_head), scratch.data_ptr(),
                    scratch.numel(), _native.stream_of(matrix))
            _native.check(status, "ct_head_loss_backward")
        if d_hidden is not None:
            d_hidden = d_hidden.to(hidden_dtype).reshape(hidden_shape)
        if d_head is not None:
            d_head = d_head.to(head_dtype)
        return d_hidden, d_head, None, None, None, None


def streamed_loss(hidden, head, weights, selection, compute_dtype, indices, values=None, log_normalizer=None,
                  temperature=1.0):
    """The loss of device tensors: hard labels `indices` [tokens, 1], or a teacher's entries."""
    if compute_dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("streamed head loss: the HIP kernels compute in bfloat16 or float32")
    _native.refuse_tangents("streamed head loss", hidden, head)
    device = hidden.device
    wide = lambda t: None if t is None else t.to(device, torch.float32).contiguous()  # noqa: E731
    tables = (indices.to(torch.int64).contiguous(), wide(values), wide(log_normalizer), wide(weights.flatten()))
    return StreamedHeadLoss.apply(hidden, head, tables, selection, compute_dtype, temperature)
