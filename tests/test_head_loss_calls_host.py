"""What the streamed losses hand to the library, on host tensors with the native calls stubbed."""

import contextlib
import types

import pytest
import torch

from causal_tuner.kernels import _native, head_loss_cuda


class _Library:
    """Records the operands of both passes."""

    def __init__(self):
        self.forward = self.backward = None

    def ct_head_loss_kept(self, *sizes):
        return 64

    def ct_head_loss_workspace(self, *sizes):
        return 64

    def ct_head_loss_forward(self, call, *rest):
        self.forward = _native.HeadLoss.from_buffer_copy(call)
        return 0

    def ct_head_loss_backward(self, call, *rest):
        self.backward = _native.HeadLoss.from_buffer_copy(call)
        self.kept = rest[1]
        return 0


@pytest.fixture
def library(monkeypatch):
    stub = _Library()
    monkeypatch.setattr(head_loss_cuda, "_native", types.SimpleNamespace(**{
        **vars(_native), "library": lambda: stub, "device_of": lambda t: contextlib.nullcontext(), "stream_of": lambda t: None}))
    return stub


def _strided(t):
    """The same values, no two of them side by side."""
    return t.new_empty(*t.shape, 2)[..., 0].copy_(t)


@pytest.mark.parametrize("restore", [torch.Tensor.contiguous, torch.clone, _strided])
@pytest.mark.parametrize("rows", [None, slice(2, 5), torch.tensor([4, 1])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_come_back_with_other_strides(dtype, rows, restore, library):
    """Pitched views that a hook on saved tensors gives back dense, or with a stride between two columns: the
    backward's addresses and pitches are those of the tensors that it has."""
    width = 16
    hidden = torch.randn(6, 40).to(dtype)[:, 8:24].requires_grad_()
    head = torch.randn(11, 48).to(dtype)[:, 16:32].requires_grad_()
    back = []

    def unpack(t):
        back.append(restore(t))
        return back[-1]
    selection = slice(0, 6) if rows is None else rows
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), unpack):
        loss = head_loss_cuda.streamed_loss(hidden, head, torch.ones(6), selection, dtype, torch.zeros(6, 1, dtype=torch.int64))
    assert library.forward.ld_hidden == 40 and library.forward.ld_head == 48
    loss.backward()
    call, size = library.backward, hidden.element_size()
    h, w = (next(t for t in back if t.shape == like.shape and t.dtype == dtype) for like in (hidden, head))
    first = selection.start if isinstance(selection, slice) else 0
    if restore is _strided:   # copies, of unit stride
        assert call.ld_hidden == call.ld_head == width
    else:
        assert (call.ld_hidden, call.ld_head) == (h.stride(0), w.stride(0)) == (width, width)
        assert call.head == w.data_ptr() and call.hidden == h.data_ptr() + first * width * size
    assert call.hidden and call.head % 16 == 0 and bool(call.rows) == isinstance(rows, torch.Tensor)
