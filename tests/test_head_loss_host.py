"""projection_loss(implementation="streamed") and distillation_loss on host tensors, and the
refusals of both."""

import math

import pytest
import torch
import torch.nn.functional as F

from causal_tuner.kernels import _native
from causal_tuner.kernels.loss import distillation_loss, projection_loss


def _inputs(rows=6, width=5, vocab=11):
    return (torch.randn(rows, width, dtype=torch.float64, requires_grad=True),
            torch.randn(vocab, width, dtype=torch.float64, requires_grad=True), torch.rand(rows) + 0.1)


def test_streamed_host_loss_is_the_host_loss():
    hidden, head = torch.randn(2, 3, 7, requires_grad=True), torch.randn(13, 7, requires_grad=True)
    targets, weights = torch.randint(13, (2, 3)), torch.tensor([[0., 1., .5], [2., 0., 1.]])
    run = lambda kind: projection_loss(hidden, head, targets, weights, compute_dtype=torch.float32,  # noqa: E731
                                       implementation=kind)
    for a, b in zip((run("streamed"), *torch.autograd.grad(run("streamed"), (hidden, head))),
                    (run("fused"), *torch.autograd.grad(run("fused"), (hidden, head)))):
        torch.testing.assert_close(a, b)


def test_one_entry_is_cross_entropy():
    hidden, head, weights = _inputs()
    labels = torch.randint(11, (6,))
    loss = distillation_loss(hidden, head, labels[:, None], torch.randn(6, 1), weights, compute_dtype=torch.float64)
    expected = (F.cross_entropy(hidden @ head.T, labels, reduction="none") * weights).sum()
    torch.testing.assert_close(loss, expected)


@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("normalizer", [False, True])
def test_entries_holes_and_equal_indices(temperature, normalizer):
    """Against kl_div over the whole vocabulary; an index outside it is no entry (whatever its value), a value of
    -inf no mass, an index given twice one with both probabilities, a row without entries no loss."""
    hidden, head, weights = _inputs()
    indices = torch.tensor([[0, 3, 5], [2, 2, 10], [-1, 4, 11], [7, 8, 9], [-1, -1, 99], [1, 1, 1]])
    values = torch.randn(6, 3, dtype=torch.float64)
    values[2, 0] = values[4, 2] = math.nan
    values[3, 1] = -math.inf
    there = (indices >= 0) & (indices < 11)
    scaled = (values / temperature).masked_fill(~there, -math.inf)
    norm = torch.logsumexp(scaled, -1) + (0.4 if normalizer else 0.0)
    q = torch.zeros(6, 11, dtype=torch.float64)
    for i in range(6):
        for k in range(3):
            if there[i, k]:
                q[i, indices[i, k]] += (scaled[i, k] - norm[i]).exp()
    loss = distillation_loss(hidden, head, indices, values, weights, temperature=temperature,
                             log_normalizer=norm.clamp_min(-50) if normalizer else None, compute_dtype=torch.float64)
    log_p = torch.log_softmax(hidden @ head.T / temperature, -1)
    expected = (F.kl_div(log_p, q, reduction="none").sum(-1) * weights).sum()
    torch.testing.assert_close(loss, expected)
    got = torch.autograd.grad(loss, (hidden, head))
    for a, b in zip(got, torch.autograd.grad(expected, (hidden, head))):
        torch.testing.assert_close(a, b)
    assert not got[0][4].any()


def test_rows_and_shapes():
    hidden, head, weights = _inputs()
    indices, values = torch.randint(11, (6, 4)), torch.randn(6, 4, dtype=torch.float64)
    run = lambda h, i, v, w, **kw: distillation_loss(h, head, i, v, w, compute_dtype=torch.float64, **kw)  # noqa: E731
    whole = run(hidden, indices, values, weights)
    folded = run(hidden.reshape(2, 3, 5), indices.reshape(2, 3, 4), values.reshape(2, 3, 4), weights.reshape(2, 3))
    torch.testing.assert_close(whole, folded)
    rows = torch.tensor([4, 1])
    torch.testing.assert_close(run(hidden, indices, values, weights, rows=rows),
                               run(hidden[rows], indices[rows], values[rows], weights[rows]))
    some = weights.clone()
    some[[0, 3]] = 0
    torch.testing.assert_close(run(hidden, indices, values, some),
                               run(hidden, indices, values, weights, rows=torch.tensor([1, 2, 4, 5])))
    assert run(hidden, indices, values, torch.zeros(6)).item() == 0


def test_refusals():
    hidden, head, weights = _inputs()
    indices, values = torch.randint(11, (6, 4)), torch.randn(6, 4)
    run = lambda *a, **kw: distillation_loss(*a, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="differ"):
        run(hidden, head, indices, values[:, :3], weights)
    with pytest.raises(ValueError, match="entries per row"):
        run(hidden, head, indices[:, :0], values[:, :0], weights)
    with pytest.raises(ValueError, match="entries per row"):
        run(hidden, head, indices.repeat(1, 257), values.repeat(1, 257), weights)
    with pytest.raises(ValueError, match="whole numbers"):
        run(hidden, head, indices.float(), values, weights)
    for temperature in (0, -1, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            run(hidden, head, indices, values, weights, temperature=temperature)
    with pytest.raises(ValueError, match="weights"):
        run(hidden, head, indices, values, weights[:5])
    with pytest.raises(ValueError, match="indices"):
        run(hidden, head, indices[:5], values[:5], weights)
    with pytest.raises(ValueError, match="log_normalizer"):
        run(hidden, head, indices, values, weights, log_normalizer=torch.zeros(5))
    with pytest.raises(ValueError, match="logits"):
        run(hidden, head[:, :4], indices, values, weights)
    with pytest.raises(ValueError, match="detach"):
        run(hidden, head, indices, values.requires_grad_(), weights)
    targets = torch.randint(11, (6,))
    with pytest.raises(ValueError, match="reuse_hidden"):
        projection_loss(hidden, head, targets, weights, implementation="streamed", reuse_hidden=True)
    with pytest.raises(ValueError, match="targets"):
        projection_loss(hidden, head, targets[:5], weights, implementation="streamed")
    with pytest.raises(ValueError, match="whole numbers"):
        projection_loss(hidden, head, targets.float(), weights, implementation="streamed")
    with pytest.raises(ValueError, match="positive"):
        projection_loss(hidden, head, targets, weights, implementation="streamed", token_budget=0)


def test_library_refuses_bad_operands_on_the_host():
    """The C entries' own checks; every call returns before anything is enqueued."""
    lib = _native.library()
    good = dict(hidden=256, head=256, indices=256, weights=256, ld_hidden=64, ld_head=64, ld_indices=1, ld_values=1,
                tokens=4, hidden_width=64, count=4, width=64, vocab=100, entries=1, dtype=_native.CT_BF16, temperature=1.0)
    forward = lambda **kw: lib.ct_head_loss_forward(_native.HeadLoss(**{**good, **kw}), 256, 1, 256, 1 << 40, 256,  # noqa: E731
                                                    1 << 40, None)
    for kw, status in [(dict(hidden=None), -1), (dict(head=264), -1), (dict(indices=None), -1), (dict(weights=None), -1),
                       (dict(count=-1), -2), (dict(width=0), -2), (dict(width=60), -2), (dict(vocab=0), -2),
                       (dict(vocab=1 << 31), -2), (dict(entries=0), -2), (dict(entries=1025, values=256), -2),
                       (dict(entries=2), -2), (dict(tokens=3), -2), (dict(ld_head=63), -2), (dict(ld_hidden=63), -2),
                       (dict(hidden_width=65), -2), (dict(temperature=0.0), -2), (dict(temperature=math.nan), -2),
                       (dict(dtype=_native.CT_F16), -3), (dict(ld_head=1 << 21), -2),
                       (dict(ld_hidden=1 << 21), -2), (dict(width=1 << 17, ld_head=1 << 17), -2), (dict(values=256, ld_values=0), -2)]:
        assert forward(**kw) == status, kw
    sizes = (4, 64, 100, 1, _native.CT_BF16)
    kept, scratch = lib.ct_head_loss_kept(*sizes, 1), lib.ct_head_loss_workspace(*sizes, 1)
    a = _native.HeadLoss(**good)
    assert kept > 0 and scratch > 0 and lib.ct_head_loss_kept(*sizes, 0) < kept
    assert lib.ct_head_loss_forward(a, 256, 1, 256, kept - 1, 256, scratch, None) == -5
    assert lib.ct_head_loss_forward(a, 256, 1, 256, kept, 256, scratch - 1, None) == -5
    assert lib.ct_head_loss_forward(a, 256, 1, 264, kept, 256, scratch, None) == -5
    assert lib.ct_head_loss_forward(a, None, 1, 256, kept, 256, scratch, None) == -1
    back = lambda **kw: lib.ct_head_loss_backward(*{**dict(  # noqa: E731
        a=a, upstream=256, kept=256, hidden_grad=1, kept_bytes=kept, d_hidden=256, ld_d_hidden=64, d_hidden_width=64,
        d_hidden_dtype=_native.CT_BF16, d_head=256, ld_d_head=64, d_head_width=64, d_head_dtype=_native.CT_BF16,
        workspace=256, workspace_bytes=0, stream=None), **kw}.values())
    assert back(upstream=None) == -1
    assert back(kept_bytes=kept - 1) == -5
    assert back(hidden_grad=0) == -5
    assert back(d_hidden_dtype=_native.CT_F16) == -3
    assert back(d_hidden_width=65) == -2
    assert back(d_hidden=None, d_head_width=65) == -2
    assert back(d_hidden=None, d_head_dtype=_native.CT_F16) == -3
    assert back(d_hidden=None) == -5
    assert lib.ct_head_loss_workspace(4, 64, 100, 1, _native.CT_F16, 1) == 0
