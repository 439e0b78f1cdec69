"""What layer_norm hands to the library, on host tensors with the native calls stubbed."""

import contextlib
import ctypes
import types

import pytest
import torch

from causal_tuner.kernels import _native, core_cuda


def _read(address, count):
    return torch.tensor((ctypes.c_float * count).from_address(address)[:])


class _Library:
    """float32 rows: y is x + 1, the statistics 2 and 3; the backward records what it is given."""

    def ct_layer_norm_backward_workspace(self, *sizes):
        return 64

    def ct_layer_norm_forward(self, x, dtype, w, bias, w_dtype, y, mean, rstd, rows, width, eps, stream):
        mean, rstd = ctypes.c_void_p(mean).value, ctypes.c_void_p(rstd).value   # as the binding's arguments
        for i, v in enumerate((ctypes.c_float * (rows * width)).from_address(x)):
            ctypes.c_float.from_address(y + 4 * i).value = v + 1
        for to, v in ((mean, 2.0), (rstd, 3.0)):
            for i in range(rows if to else 0):
                ctypes.c_float.from_address(to + 4 * i).value = v
        return 0

    def ct_layer_norm_backward(self, x, dtype, w, w_dtype, mean, rstd, dy, dx, dw, dbias, rows, width, *rest):
        self.x, self.w = _read(x, rows * width).reshape(rows, width), _read(w, width)
        self.stats = _read(mean, rows), _read(rstd, rows)
        self.dy = _read(dy, rows * width).reshape(rows, width)
        return 0


@pytest.fixture
def library(monkeypatch):
    stub = _Library()
    monkeypatch.setattr(core_cuda, "_native", types.SimpleNamespace(**{
        **vars(_native), "library": lambda: stub, "device_of": lambda t: contextlib.nullcontext(), "stream_of": lambda t: None}))
    return stub


def _strided(t):
    """The same values, no two of them side by side."""
    return t.new_full((*t.shape, 2), 9.0)[..., 0].copy_(t)


def test_saved_tensors_come_back_with_other_strides(library):
    x, weight = torch.randn(5, 6, requires_grad=True), torch.randn(6, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _strided):
        y = core_cuda.layer_norm_device(x, weight, None, 1e-5)
    dy = torch.randn(5, 6)
    y.backward(dy)
    assert torch.equal(library.x, x.detach()) and torch.equal(library.w, weight.detach()) and torch.equal(library.dy, dy)
    assert torch.equal(library.stats[0], torch.full((5,), 2.0)) and torch.equal(library.stats[1], torch.full((5,), 3.0))


@pytest.mark.parametrize("no_grad", [False, True])
def test_a_trace_records_the_call(no_grad, library):
    """Without gradients too: a traced function computes from its new input, it does not return unwritten memory."""
    with torch.set_grad_enabled(not no_grad):
        traced = torch.jit.trace(lambda x: core_cuda.layer_norm_device(x, None, None, 1e-5), (torch.zeros(3, 4),),
                                 check_trace=False)
        for _ in range(2):
            x = torch.randn(3, 4)
            assert torch.equal(traced(x), x + 1)
