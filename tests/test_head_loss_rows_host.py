"""The `rows` of the streamed losses on host tensors: what the numbers mean is what they mean on the device."""

import pytest
import torch

from causal_tuner.kernels.loss import distillation_loss, projection_loss

F32 = torch.float32


def _calls(tokens=6, width=5, vocab=11):
    hidden, head = torch.randn(tokens, width, requires_grad=True), torch.randn(vocab, width, requires_grad=True)
    weights, labels = torch.rand(tokens) + 0.1, torch.randint(vocab, (tokens,))
    indices, values = torch.randint(vocab, (tokens, 3)), torch.randn(tokens, 3)
    calls = [lambda w, rows: projection_loss(hidden, head, labels, w, implementation="streamed", compute_dtype=F32, rows=rows),
             lambda w, rows: distillation_loss(hidden, head, indices, values, w, compute_dtype=F32, rows=rows)]
    return hidden, head, weights, calls


@pytest.mark.parametrize("which", [0, 1])
def test_numbers_outside_the_batch_have_no_loss(which):
    hidden, head, weights, calls = _calls()
    got = calls[which](weights, torch.tensor([3, 6, 0, -1, 1 << 40, -6]))
    want = calls[which](weights, torch.tensor([3, 0]))
    torch.testing.assert_close(got, want, rtol=0, atol=0)
    for a, b in zip(torch.autograd.grad(got, (hidden, head)), torch.autograd.grad(want, (hidden, head))):
        torch.testing.assert_close(a, b, rtol=0, atol=0)


@pytest.mark.parametrize("which", [0, 1])
def test_rows_given_twice_count_twice(which):
    hidden, head, weights, calls = _calls()
    got = calls[which](weights, torch.tensor([3, 0, 3, 5, 3, 0]))
    want = calls[which](weights * torch.tensor([2., 0., 0., 3., 0., 1.]), None)
    torch.testing.assert_close(got, want)
    for a, b in zip(torch.autograd.grad(got, (hidden, head)), torch.autograd.grad(want, (hidden, head))):
        torch.testing.assert_close(a, b)


@pytest.mark.parametrize("tokens", [1, 6])
@pytest.mark.parametrize("which", [0, 1])
def test_masks_and_lists(which, tokens):
    hidden, head, weights, calls = _calls(tokens)
    numbers = [0] if tokens == 1 else [1, 3, 4]
    mask = torch.zeros(tokens, dtype=torch.bool)
    mask[numbers] = True
    want = calls[which](weights, torch.tensor(numbers))
    for rows in (mask, numbers):
        got = calls[which](weights, rows)
        torch.testing.assert_close(got, want, rtol=0, atol=0)
        for a, b in zip(torch.autograd.grad(got, (hidden, head)), torch.autograd.grad(want, (hidden, head), retain_graph=True)):
            torch.testing.assert_close(a, b, rtol=0, atol=0)


@pytest.mark.parametrize("rows", [[], torch.zeros(0, dtype=torch.int64), torch.tensor([-1, 9])])
@pytest.mark.parametrize("which", [0, 1])
def test_no_rows(which, rows):
    hidden, head, weights, calls = _calls()
    loss = calls[which](weights, rows)
    dh, dw = torch.autograd.grad(loss, (hidden, head))
    assert loss.item() == 0 and not dh.any() and not dw.any()
