"""What the streamed losses hand to the library, on host tensors with the native calls stubbed."""

import contextlib
import types

import pytest
import torch
from torch.autograd import forward_ad

from causal_tuner.kernels import _native, head_loss_cuda
from causal_tuner.kernels.loss import distillation_loss, projection_loss


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


@pytest.mark.parametrize("rows,refused", [((1 << 22) - 64, False), ((1 << 22) - 63, True)])
def test_rows_of_a_head_gradient(rows, refused, library):
    """More rows than a tile's offsets reach are refused by name before anything is laid out; a frozen head takes them."""
    hidden, head = torch.zeros(1, 8).expand(rows, 8).requires_grad_(), torch.zeros(3, 8, requires_grad=True)
    run = lambda w: head_loss_cuda.streamed_loss(hidden, w, torch.ones(1).expand(rows), slice(0, rows), torch.float32,  # noqa: E731
                                                 torch.zeros(1, 1, dtype=torch.int64).expand(rows, 1))
    if refused:
        with pytest.raises(ValueError, match="head's gradient"):
            run(head)
        assert library.forward is None
        run(head.detach())
    else:
        run(head)
    assert library.forward.count == rows


def test_library_refuses_a_head_gradient_of_more_rows():
    lib = _native.library()
    rows = (1 << 22) - 63
    a = _native.HeadLoss(hidden=256, head=256, ld_hidden=64, ld_head=64, tokens=rows, hidden_width=64, count=rows, width=64,
                         vocab=100, entries=1, dtype=_native.CT_BF16, temperature=1.0)
    back = lambda d_hidden, d_head: lib.ct_head_loss_backward(a, 256, None, 1, 0, d_hidden, 64, 64, _native.CT_BF16, d_head, 64,  # noqa: E731
                                                              64, _native.CT_BF16, 256, 1 << 40, None)
    assert back(None, 256) == back(256, 256) == -2
    assert back(256, None) == -5   # only the missing buffer
    a.count -= 1
    assert back(None, 256) == -5
    sizes = (64, 100, 1, _native.CT_BF16, 2)
    assert lib.ct_head_loss_workspace(rows, *sizes) == 0 < lib.ct_head_loss_workspace(rows - 1, *sizes)


def test_weights_that_ask_for_a_gradient_are_refused():
    """On the host as on the device, where none is made: nothing is dropped without a word."""
    hidden, head, weights = torch.randn(4, 8, requires_grad=True), torch.randn(9, 8), torch.rand(4, requires_grad=True)
    indices, labels = torch.randint(9, (4, 3)), torch.randint(9, (4,))
    calls = [lambda w: distillation_loss(hidden, head, indices, torch.randn(4, 3), w),
             lambda w: projection_loss(hidden, head, labels, w, implementation="streamed")]
    for call in calls:
        with pytest.raises(ValueError, match="weights get no gradient"):
            call(weights)
        call(weights.detach())
        with torch.no_grad():
            call(weights)


@pytest.mark.parametrize("which", ["hidden", "head", "weights", "values", "log_normalizer"])
def test_forward_derivatives_are_refused(which, library):
    given = dict(hidden=torch.randn(4, 8), head=torch.randn(9, 8), weights=torch.rand(4), values=torch.randn(4, 3),
                 log_normalizer=torch.zeros(4))

    def run(t):
        return head_loss_cuda.streamed_loss(t["hidden"], t["head"], t["weights"], slice(0, 4), torch.float32,
                                            torch.randint(9, (4, 3)), t["values"], t["log_normalizer"])
    with forward_ad.dual_level():
        run(given)
        given[which] = forward_ad.make_dual(given[which], torch.ones_like(given[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            run(given)
