"""The end of a training step as it is used: final layer norm, streamed cross-entropy plus distillation
from a teacher's top logits, and their backward in one pass; the decoder's losses on the same operators."""

import pytest
import torch

from head_loss_reference import targets

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _float64(x, weight, bias, head, labels, indices, values, weights, temperature, alpha):
    mean = x.mean(-1, keepdim=True)
    h = (x - mean) * ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt() * weight + bias
    logits = h @ head.T
    hard = -torch.log_softmax(logits, -1).gather(1, labels[:, None])[:, 0]
    q = targets(indices, values, temperature, None, len(head))
    soft = torch.where(q > 0, q * (q.clamp_min(1e-300).log() - torch.log_softmax(logits / temperature, -1)), 0).sum(-1)
    return (weights.double() * ((1 - alpha) * hard + alpha * temperature ** 2 * soft)).sum()


@pytest.mark.parametrize("dtype,tolerance", [(torch.float32, 2e-5), (torch.bfloat16, 2e-2)])
def test_norm_and_both_losses(dtype, tolerance):
    """Against float64 through autograd. bf16: the norm's output and its incoming gradients are rounded
    (2^-8 each, twice for the sum of two losses' gradients), so norms of errors stay below 5 x 2^-8."""
    from causal_tuner.kernels.loss import distillation_loss, projection_loss
    from causal_tuner.modeling.norm import LayerNorm
    rows, width, vocab, temperature, alpha = 300, 192, 2500, 2.0, 0.4
    x = (torch.randn(1, rows, width, device="cuda") + 0.3).to(dtype).requires_grad_()
    norm = LayerNorm(width, EPS, dtype, "cuda")
    head = (torch.randn(vocab, width, device="cuda") * 0.15).to(dtype).requires_grad_()
    labels = torch.randint(vocab, (1, rows), device="cuda")
    weights = (torch.rand(1, rows, device="cuda") > 0.3).float() / rows
    values, indices = (torch.randn(1, rows, vocab, device="cuda") * 2).topk(20, -1)
    hidden = norm(x)
    loss = projection_loss(hidden, head, labels, weights * (1 - alpha), implementation="streamed", compute_dtype=dtype) \
        + distillation_loss(hidden, head, indices, values, weights * (alpha * temperature ** 2), temperature=temperature,
                            compute_dtype=dtype)
    leaves = (x, norm.weight, norm.bias, head)
    grads = torch.autograd.grad(loss, leaves)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = _float64(wide[0][0], wide[1], wide[2], wide[3], labels[0], indices[0], values[0], weights[0], temperature, alpha)
    assert abs(loss.item() - want.item()) <= tolerance * abs(want.item())
    for got, exact in zip(grads, torch.autograd.grad(want, wide)):
        assert (got.double() - exact).norm() <= tolerance * exact.norm()


def _tiny(norm):
    from causal_tuner.modeling.decoder import Decoder, DecoderConfig
    config = DecoderConfig(hidden_size=128, num_attention_heads=2, head_dim=64, intermediate_size=256,
                           num_hidden_layers=2, vocab_size=300, attention="packed", norm=norm)
    torch.manual_seed(5)
    model = Decoder(config, rank=8, device="cuda")
    for name, p in model.named_parameters():
        if "lora_B" in name:
            torch.nn.init.normal_(p, std=0.1)
    model.install_nf4()
    return model


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_decoder_losses(norm):
    """The streamed loss against the fused one on the same hidden states: the fused path rounds its
    logits (of size 1 here) to bf16, the streamed one does not, so the adapters' gradients agree to a
    few of those roundings; distillation from one certain entry per row is the loss of that label."""
    model = _tiny(norm)
    records = [(0, 40), (40, 70)]
    ids = torch.randint(300, (1, 70), device="cuda")
    labels = torch.randint(300, (1, 70), device="cuda")
    weights = (torch.rand(1, 70, device="cuda") > 0.4).float() / 40
    leaves = [p for p in model.parameters() if p.requires_grad]
    losses = [model.loss(ids, labels, weights, records), model.loss(ids, labels, weights, records, implementation="streamed"),
              model.distillation_loss(ids, labels[..., None], torch.zeros(1, 70, 1, device="cuda"), weights, records)]
    grads = [torch.autograd.grad(loss, leaves) for loss in losses]
    assert abs(losses[1].item() - losses[0].item()) <= 2e-3 * losses[0].item()
    for fused, streamed, distilled in zip(*grads):
        assert torch.isfinite(streamed).all() and streamed.any()
        assert (streamed - fused).norm() <= 2e-2 * fused.norm()
        assert torch.equal(streamed, distilled)
