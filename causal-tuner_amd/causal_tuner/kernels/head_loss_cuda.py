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


_MAX_PITCH = 1 << 20     # elements between two rows
_MAX_WIDTH = 1 << 16
_MAX_VOCAB = (1 << 31) - 1024
_MAX_ROWS = (1 << 24) - 256
_MAX_VALUES = (1 << 35) - 256    # of the padded rows
_MAX_HEAD_ROWS = (1 << 22) - 64  # with the head's gradient


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


def _plain(t):
    """Whether t's rows have unit stride and a pitch that the kernels take."""
    return t.stride(1) == 1 and t.shape[1] <= t.stride(0) <= _MAX_PITCH


def _aligned_head(head):
    """`head` with unit-stride rows that start at 16-byte boundaries, bf16 widths a multiple of 8:
    itself, or a copy padded with zeros."""
    if head.dtype == torch.bfloat16:
        pad = -head.shape[1] % 8
        if pad:
            return torch.nn.functional.pad(head, (0, pad))
        if head.stride(0) % 8 or head.data_ptr() % 16:
            return head.clone(memory_format=torch.contiguous_format)
    return head if _plain(head) else head.clone(memory_format=torch.contiguous_format)


def _plain_rows(hidden):
    h = hidden.reshape(-1, hidden.shape[-1])
    return h if _plain(h) else h.clone(memory_format=torch.contiguous_format)


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


class StreamedHeadLoss(torch.autograd.Function):
    """What the backward needs besides the tensors is worked out in the forward: the backward runs on
    autograd's device thread, where Python is several times slower."""

    @staticmethod
    def forward(ctx, hidden, head, tables, selection, compute_dtype, temperature):
        need_hidden, need_head = ctx.needs_input_grad[:2]
        indices, values, normalizer, weights = tables
        tokens, device, entries = len(indices), hidden.device, indices.shape[1]
        first, rows, count = _rows_of(selection, tokens, device)
        matrix = _aligned_head(head.to(compute_dtype))
        vocab, width = matrix.shape
        if need_head and count > _MAX_HEAD_ROWS:
            raise ValueError(f"streamed head loss: {count} rows; the HIP kernels take up to {_MAX_HEAD_ROWS} at once with the "
                             "head's gradient")
        if count > _MAX_ROWS or (count + 255) // 256 * 256 * ((width + 63) // 64 * 64) > _MAX_VALUES:
            raise ValueError(f"streamed head loss: {count} rows of {width} values; the HIP kernels take up to {_MAX_ROWS} rows "
                             f"and {_MAX_VALUES} values at once")
        h = _plain_rows(hidden.to(compute_dtype))
        skip = first * entries
        ld, code = h.stride(0), _native.dtype_code(compute_dtype)
        call = _native.HeadLoss(
            h.data_ptr() + first * ld * h.element_size(), matrix.data_ptr(), _native.ptr(rows),
            indices.data_ptr() + 8 * skip, None if values is None else values.data_ptr() + 4 * skip,
            None if normalizer is None else normalizer.data_ptr() + 4 * first, weights.data_ptr() + 4 * first,
            max(ld, h.shape[1]), matrix.stride(0), entries, entries, tokens - first, h.shape[1], count, width, vocab,
            entries, code, temperature)
        lib, sizes, sums = _native.library(), (count, width, vocab, entries, code), int(need_hidden)
        loss = torch.empty((), dtype=torch.float32, device=device)
        kept_bytes = lib.ct_head_loss_kept(*sizes, sums)
        kept = _workspace(kept_bytes, device)
        scratch = _workspace(lib.ct_head_loss_workspace(*sizes, sums), device)
        with _native.device_of(h):
            status = lib.ct_head_loss_forward(call, loss.data_ptr(), sums, kept.data_ptr(), kept_bytes, scratch.data_ptr(),
                                              scratch.numel(), _native.stream_of(h))
        _native.check(status, "ct_head_loss_forward")
        if need_hidden or need_head:
            ctx.save_for_backward(h if need_head else None, matrix, kept, rows)
            d_hidden = (hidden.shape, hidden.dtype, rows is None and count == tokens)
            d_head = (head.shape, head.dtype, lib.ct_head_loss_workspace(*sizes, 2)) if need_head else None
            # the targets are in what is kept
            call.indices = call.values = call.log_normalizer = call.weights = None
            ctx.plan = (lib.ct_head_loss_backward, call, first, count, sums, kept_bytes, code, d_hidden, d_head,
                        (matrix.stride(), h.stride()))
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        h, matrix, kept, rows = ctx.saved_tensors
        backward, call, first, count, sums, kept_bytes, code, hidden_plan, head_plan, strides = ctx.plan
        _native.refuse_tangents("streamed head loss", upstream)
        need_hidden, need_head = ctx.needs_input_grad[:2]
        device = matrix.device
        d_hidden = d_head = scratch = None
        hidden_at = head_at = scratch_at = None
        width = hidden_code = head_code = scratch_bytes = 0
        if need_hidden:
            shape, dtype, whole = hidden_plan
            width = shape[-1]
            wide = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
            d_hidden = (torch.empty if whole else torch.zeros)(shape, dtype=wide, device=device)
            hidden_code = _native.dtype_code(wide)
            hidden_at = d_hidden.data_ptr() + first * width * d_hidden.element_size()
        if need_head:
            shape, head_dtype, scratch_bytes = head_plan
            width = shape[1]
            wide = torch.bfloat16 if code == _native.CT_BF16 and head_dtype == torch.bfloat16 else torch.float32
            d_head = (torch.empty if count else torch.zeros)(shape, dtype=wide, device=device)
            head_code, head_at = _native.dtype_code(wide), d_head.data_ptr()
            scratch = _workspace(scratch_bytes, device)
            scratch_at = scratch.data_ptr()
        if count:
            call, head_in = _native.HeadLoss.from_buffer_copy(call), matrix.data_ptr()
            # hooks on saved tensors (save_on_cpu) may have brought one back in another place and with other strides
            if (matrix.stride() != strides[0] or head_in % 16 or (h is not None and h.stride() != strides[1])
                    or kept.stride(0) != 1 or (rows is not None and rows.stride(0) != 1)):
                matrix, kept = _aligned_head(matrix), kept.contiguous()
                head_in, call.ld_head = matrix.data_ptr(), matrix.stride(0)
                if h is not None:
                    h = _plain_rows(h)
                    call.ld_hidden = max(h.stride(0), h.shape[1])
                rows = None if rows is None else rows.contiguous()
            call.head, call.rows = head_in, _native.ptr(rows)
            if h is not None:
                call.hidden = h.data_ptr() + first * h.stride(0) * h.element_size()
            # autograd has made the tensors' device current
            status = backward(call, upstream.to(torch.float32).data_ptr(), kept.data_ptr(), sums, kept_bytes, hidden_at, width,
                              width, hidden_code, head_at, width, width, head_code, scratch_at, scratch_bytes,
                              _native.stream_of(matrix))
            if status:
                _native.check(status, "ct_head_loss_backward")
        if need_hidden and d_hidden.dtype != hidden_plan[1]:
            d_hidden = d_hidden.to(hidden_plan[1])
        if need_head and d_head.dtype != head_dtype:
            d_head = d_head.to(head_dtype)
        return d_hidden, d_head, None, None, None, None


def streamed_loss(hidden, head, weights, selection, compute_dtype, indices, values=None, log_normalizer=None,
                  temperature=1.0):
    """The loss of device tensors: hard labels `indices` [tokens, 1], or a teacher's entries."""
    if compute_dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("streamed head loss: the HIP kernels compute in bfloat16 or float32")
    if head.shape[1] > _MAX_WIDTH or len(head) > _MAX_VOCAB:
        raise ValueError(f"streamed head loss: head {tuple(head.shape)}; the HIP kernels take up to {_MAX_VOCAB} entries and "
                         f"a width of {_MAX_WIDTH}")
    _native.refuse_tangents("streamed head loss", hidden, head, weights, values, log_normalizer)
    device = hidden.device
    wide = lambda t: None if t is None else t.to(device, torch.float32).contiguous()  # noqa: E731
    tables = (indices.to(torch.int64).contiguous(), wide(values), wide(log_normalizer), wide(weights.flatten()))
    return StreamedHeadLoss.apply(hidden, head, tables, selection, compute_dtype, temperature)
