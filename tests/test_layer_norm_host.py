"""layer_norm and LayerNorm on host tensors, and their refusals."""

import pytest
import torch

from causal_tuner.kernels import _native
from causal_tuner.modeling.decoder import Decoder, DecoderConfig
from causal_tuner.modeling.norm import LayerNorm, layer_norm


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_host_formula(weight, bias):
    x = torch.randn(2, 3, 7, dtype=torch.float64, requires_grad=True)
    w = torch.randn(7, dtype=torch.float64, requires_grad=True) if weight else None
    b = torch.randn(7, dtype=torch.float64, requires_grad=True) if bias else None
    y, want = layer_norm(x, w, b, 1e-3), torch.nn.functional.layer_norm(x, (7,), w, b, 1e-3)
    torch.testing.assert_close(y, want)
    leaves = [t for t in (x, w, b) if t is not None]
    dy = torch.randn_like(y)
    for got, grad in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        torch.testing.assert_close(got, grad)


def test_module():
    norm = LayerNorm(6, 1e-5, torch.bfloat16, "cpu")
    x = torch.randn(4, 6).bfloat16()
    assert norm(x).dtype == torch.bfloat16 and torch.equal(norm(x), layer_norm(x, norm.weight, norm.bias, 1e-5))
    assert LayerNorm(6, 1e-5, torch.float32, "cpu", bias=False).bias is None


def test_refusals():
    x, w = torch.randn(3, 4), torch.ones(4)
    with pytest.raises(ValueError, match="weight"):
        layer_norm(x, torch.ones(3))
    with pytest.raises(ValueError, match="bias"):
        layer_norm(x, w, torch.ones(1, 4))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, w, eps=-1)
    with pytest.raises(ValueError, match="floating"):
        layer_norm(torch.ones(3, 4, dtype=torch.int64), w)
    for empty in (torch.zeros(3, 0), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="width"):
            layer_norm(empty)


def test_decoder_norms():
    config = DecoderConfig(hidden_size=32, num_attention_heads=2, head_dim=16, intermediate_size=48, num_hidden_layers=1,
                           vocab_size=50, norm="layer")
    model = Decoder(config, rank=4)
    assert isinstance(model.norm, LayerNorm) and isinstance(model.layers[0].input_layernorm, LayerNorm)
    assert not any(p.requires_grad for n, p in model.named_parameters() if "norm" in n)
    with pytest.raises(ValueError, match="norm"):
        DecoderConfig(norm="batch")


def test_library_refuses_bad_operands_on_the_host():
    lib = _native.library()
    bf16 = _native.CT_BF16
    forward = lambda *a: lib.ct_layer_norm_forward(*a, None)  # noqa: E731
    assert forward(None, bf16, None, None, bf16, 256, None, None, 2, 8, 1e-5) == -1
    assert forward(256, bf16, None, None, bf16, 256, 256, None, 2, 8, 1e-5) == -1
    assert forward(256, 7, None, None, bf16, 256, None, None, 2, 8, 1e-5) == -3
    assert forward(256, bf16, 256, None, 7, 256, None, None, 2, 8, 1e-5) == -3
    assert forward(256, bf16, None, None, bf16, 256, None, None, 2, 0, 1e-5) == -2
    assert forward(256, bf16, None, None, bf16, 256, None, None, -1, 8, 1e-5) == -2
    assert forward(256, bf16, None, None, bf16, 256, None, None, 2, 8, -1.0) == -2
    need = lib.ct_layer_norm_backward_workspace(2, 8, bf16, 1)
    assert need > 0 and lib.ct_layer_norm_backward_workspace(2, 8, bf16, 0) == 0
    backward = lambda *a: lib.ct_layer_norm_backward(*a, None)  # noqa: E731
    assert backward(256, bf16, 256, bf16, 256, 256, 256, 256, 256, 256, 2, 8, None, need) == -5
    assert backward(256, bf16, 256, bf16, 256, 256, 256, 256, 256, 256, 2, 8, 256, need - 1) == -5
    assert backward(256, bf16, 256, bf16, None, 256, 256, 256, 256, 256, 2, 8, 256, need) == -1
    assert backward(256, bf16, 256, bf16, 256, 256, 256, 256, 256, 256, 2, 0, 256, need) == -2
