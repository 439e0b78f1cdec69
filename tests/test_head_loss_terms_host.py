"""The bounds for two bf16 terms take two terms and refuse one, on the host."""

import pytest
import torch

from head_loss_terms import expected, inputs


def _terms(x, count):
    """x as the sum of `count` bf16 values."""
    held = torch.zeros_like(x)
    for _ in range(count):
        held = held + (x - held).to(torch.bfloat16).double()
    return held


@pytest.mark.parametrize("rows,width,offset", [(1, 16, 0.0), (64, 16, 0.0), (65, 16, 33.0), (128, 16, 33.0), (128, 1032, 0.0), (17, 16, 33.0), (256, 16, 0.0)])
@pytest.mark.parametrize("count", [1, 2])
def test_one_term_is_refused(count, rows, width, offset):
    hidden, head, labels, weights = inputs(rows, width, offset, "cpu")
    want, b_dh, b_dw = expected(hidden, head, labels, weights)
    h, w, c, logits, q, mass, lse, p, d = want[3]
    e = _terms(torch.where(q > 0, 0.0, p), count)            # the targets' own terms are apart
    dh = (c[:, None] * torch.where(q > 0, 0.0, e)) @ w + torch.where(q > 0, d, 0.0) @ w
    dw = _terms(d, count).T @ h
    for got, exact, bound in ((dh, want[1], b_dh), (dw, want[2], b_dw)):
        worst = ((got - exact).abs() / bound).max()
        assert worst <= 1 if count == 2 else worst > 1.5, worst
