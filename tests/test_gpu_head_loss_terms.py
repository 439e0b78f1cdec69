"""Few rows of the streamed loss in bf16: the exponentials behind the hidden gradient of up to 128 rows and the derivative
behind the head's of up to 256 are held in two bf16 terms."""

import pytest
import torch

from head_loss_reference import check
from head_loss_terms import COLUMNS, expected, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0.0, 33.0])
@pytest.mark.parametrize("width", [16, 1032])   # 1032: the logits in chunks of their reduction, through memory
@pytest.mark.parametrize("rows", [1, 17, 64, 65, 127, 128, 129, 255, 256])
def test_two_terms(rows, width, offset):
    from causal_tuner.kernels.loss import projection_loss
    hidden, head, labels, weights = inputs(rows, width, offset, "cuda")
    hidden.requires_grad_()
    head.requires_grad_()
    loss = projection_loss(hidden, head, labels, weights, implementation="streamed")
    dh, dw = torch.autograd.grad(loss, (hidden, head))
    assert dh.dtype == dw.dtype == torch.float32
    want, b_dh, b_dw = expected(hidden, head, labels, weights)
    assert not dh[:, COLUMNS:].any() and not dw[:, COLUMNS:].any()
    if rows <= 128:
        check("dh", dh[:, :COLUMNS], want[1], b_dh)
    check("dW", dw[:, :COLUMNS], want[2], b_dw)
