"""Calls of layer norm beside those of a plain training step."""

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _backward(x, weight, stats, dy, dx, dw, db):
    from causal_tuner.kernels import _native
    rows, width = x.shape
    lib, code = _native.library(), _native.dtype_code(x.dtype)
    workspace = torch.empty(lib.ct_layer_norm_backward_workspace(rows, width, code, 1), dtype=torch.uint8, device="cuda")
    with _native.device_of(x):
        _native.check(lib.ct_layer_norm_backward(
            x.data_ptr(), code, weight.data_ptr(), _native.dtype_code(weight.dtype), stats.data_ptr(),
            stats.data_ptr() + 4 * rows, dy.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, width,
            workspace.data_ptr(), workspace.numel(), _native.stream_of(x)), "ct_layer_norm_backward")


@pytest.mark.parametrize("dtype,width", [(F32, 8), (BF16, 1023), (F32, 1023), (F32, 4096), (BF16, 8192), (F32, 8196), (F32, 12288),
                                         (BF16, 16392), (F16, 20001), (F32, 20001)])
def test_input_gradient_over_the_incoming_one(width, dtype):
    """dx may be dy itself, in rows that registers hold and in wider ones: the same bits as apart."""
    rows, g = 70, torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, dy, weight = make(rows, width).to(dtype), make(rows, width).to(dtype), make(width)
    mean, var = x.float().mean(-1), x.float().var(-1, unbiased=False)
    stats = torch.stack([mean, (var + 1e-5).rsqrt()])
    apart, over = [(torch.empty_like(dy), torch.empty(width, device="cuda"), torch.empty(width, device="cuda")) for _ in range(2)]
    _backward(x, weight, stats, dy, *apart)
    incoming = dy.clone()
    _backward(x, weight, stats, incoming, incoming, *over[1:])
    for name, a, b in zip(("dx", "dw", "db"), (incoming, *over[1:]), apart):
        assert torch.equal(a, b), name
    # rows 2^-24 each, of sums of magnitudes of about 70 (dbias) in any order
    assert (apart[2] - dy.double().sum(0)).abs().max() <= rows * 2.0 ** -24 * dy.double().abs().sum(0).max()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grads", [False, True])
def test_traced_calls(grads):
    """A trace holds the call itself: new inputs, of other row counts too, with and without gradients."""
    from causal_tuner.modeling.norm import LayerNorm
    norm = LayerNorm(72, 1e-5, BF16, "cuda").requires_grad_(grads)
    make = lambda n: torch.randn(n, 72, device="cuda").to(BF16).requires_grad_(grads)  # noqa: E731
    with torch.set_grad_enabled(grads):
        traced = torch.jit.trace(norm, (make(5),), check_trace=False)
        for n in (5, 5, 9):
            x = make(n)
            got, want = traced(x), norm(x)
            assert torch.equal(got, want)
            if grads:
                dy, leaves = torch.randn_like(want), (x, norm.weight, norm.bias)
                for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
                    assert torch.equal(a, b)
