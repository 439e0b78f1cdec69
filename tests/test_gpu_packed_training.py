"""The packed attention kernels and FusedMuon as a training step uses them: the decoder with
attention="packed" against the same model in float32 torch on the host and against its own
SDPA path, and Muon steps over its adapters against the iteration in float64."""

import pytest
import torch

from test_gpu_decoder import _host_loss
from test_gpu_muon import A, E32, _reference

pytestmark = pytest.mark.gpu

RECORDS = [(0, 37), (37, 100), (100, 161)]


def _model(attention):
    from causal_tuner.modeling.decoder import Decoder, DecoderConfig
    config = DecoderConfig(hidden_size=128, num_attention_heads=2, head_dim=64, intermediate_size=256,
                           num_hidden_layers=2, vocab_size=300, attention=attention)
    torch.manual_seed(5)
    model = Decoder(config, rank=8, device="cuda")
    for name, p in model.named_parameters():
        if "lora_B" in name:
            torch.nn.init.normal_(p, std=0.1)
    model.install_nf4()
    return model


def _batch():
    g = torch.Generator().manual_seed(3)
    ids, targets = (torch.randint(300, (161,), generator=g).cuda() for _ in range(2))
    weights = (torch.rand(161, generator=g) > 0.2).float().cuda()
    return ids[None], targets[None], weights[None]


def _gradients(model, records):
    ids, targets, weights = _batch()
    model.zero_grad(set_to_none=True)
    loss = model.loss(ids, targets, weights, records)
    loss.backward()
    return loss.item(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


def test_packed_decoder_step():
    """Loss within 2e-2 of the float32 host model and every adapter's gradient within 5e-2 in
    norm, the bars of the SDPA path; bit-identical when repeated, also with a layout made ahead."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    model = _model("packed")
    loss, grads = _gradients(model, RECORDS)
    ids, targets, weights = _batch()
    want, leaves = _host_loss(model, ids[0], targets[0], weights[0], RECORDS)
    want.backward()
    assert abs(loss - want.item()) <= 2e-2 * abs(want.item())
    assert set(grads) == set(leaves)
    for name, grad in grads.items():
        reference = leaves[name].grad
        assert (grad.cpu() - reference).norm() <= 5e-2 * reference.norm(), name
    again, same = _gradients(model, AttentionLayout(RECORDS, "cuda"))
    assert again == loss and all(torch.equal(grads[n], same[n]) for n in grads)
    sdpa, theirs = _gradients(_model("sdpa"), RECORDS)
    assert abs(loss - sdpa) <= 2e-2 * abs(sdpa)
    with pytest.raises(ValueError):   # records that leave tokens out
        model.loss(ids, targets, weights, [(0, 37), (37, 100)])


def test_muon_steps_of_a_decoder():
    """Two steps of the packed decoder's adapters: each parameter against the update computed in
    float64 from its gradient and momentum (test_gpu_muon.py gives the bounds)."""
    from causal_tuner.optim import FusedMuon
    model = _model("packed")
    names, params = zip(*[(n, p) for n, p in model.named_parameters() if p.requires_grad])
    optimizer = FusedMuon(params, lr=0.02, weight_decay=0.1, momentum=0.95)
    momentum = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    for _ in range(2):
        _gradients(model, RECORDS)
        before = [p.detach().double() for p in params]
        optimizer.step()
        for name, p, old, m in zip(names, params, before, momentum):
            m.mul_(0.95).add_(p.grad.double(), alpha=0.05)
            buffer = optimizer.state[p]["momentum_buffer"]
            assert ((buffer.double() - m).abs() <= 8 * E32 * (m.abs() + p.grad.abs().max())).all(), name
            m.copy_(buffer)
            direction, bound = _reference(0.95 * m + 0.05 * p.grad.double())
            factor = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            want = old * (1 - 0.02 * 0.1) - factor * direction
            allowed = factor * (bound + 3 * E32 * A ** 5 + 4 * E32 * direction.abs()) + 5 * E32 * old.abs()
            over = (p.double() - want).abs() - allowed
            assert over.max() <= 0, f"{name}: {over.max()} over"
