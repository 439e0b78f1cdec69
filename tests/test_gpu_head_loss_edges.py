"""Calls of the streamed losses beside those of a plain training step: hooks on saved tensors, rows given
twice, operands that must not be dropped."""

import pytest
import torch

from head_loss_reference import bounds, check, reference

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _pitched(rows, width, pitch, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn(rows, pitch, device="cuda", generator=g).to(dtype)
    return wide[:, 8:8 + width].requires_grad_()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("frozen", [False, True])
def test_saved_on_the_host(frozen, rows, dtype):
    """Pitched views come back from save_on_cpu as dense ones, and the gradients are those of the views."""
    from causal_tuner.kernels.loss import projection_loss
    hidden, head = _pitched(rows, 72, 100 if dtype == F32 else 104, dtype, 1), _pitched(777, 72, 136, dtype, 2)
    head.requires_grad_(not frozen)
    labels = torch.randint(777, (rows,), device="cuda")
    weights = torch.rand(rows, device="cuda") + 0.1
    leaves = [t for t in (hidden, head) if t.requires_grad]

    def step():
        loss = projection_loss(hidden, head, labels, weights, implementation="streamed", compute_dtype=dtype)
        return loss
    want = torch.autograd.grad(step(), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = step()
    for a, b in zip(torch.autograd.grad(loss, leaves), want):
        assert torch.equal(a, b)


def test_float32_head_gradient_of_very_many_rows():
    """26992 steps of 64 rows: the first count whose last step a rounded reciprocal puts into a product of terms
    that there is not. All rows but the last 64 are zero, so that the head's gradient is theirs."""
    from causal_tuner.kernels.loss import projection_loss
    rows, width, vocab = 26992 * 64, 72, 130
    g = torch.Generator(device="cuda").manual_seed(1)
    hidden = torch.zeros(rows, width, device="cuda")
    hidden[-64:] = torch.randn(64, width, device="cuda", generator=g)
    head = (torch.randn(vocab, width, device="cuda", generator=g) * 0.2).requires_grad_()
    labels = torch.randint(vocab, (rows,), device="cuda", generator=g)
    weights = torch.ones(rows, device="cuda")
    loss = projection_loss(hidden, head, labels, weights, implementation="streamed", compute_dtype=F32, rows=slice(0, rows))
    dw, = torch.autograd.grad(loss, head)
    h = hidden[-64:].double()
    d = torch.softmax(h @ head.detach().double().T, -1)
    d[torch.arange(64), labels[-64:]] -= 1
    # float32 throughout: a derivative within 2^-17 of its size and 2^-20 (a probability's error and the target's),
    # then 64 products and sums
    bound = (d.abs() * 2.0 ** -17 + 2.0 ** -20).T @ h.abs() * (1 + 64 * 2.0 ** -24)
    assert ((dw.double() - d.T @ h).abs() <= bound).all()


def test_head_gradient_of_the_most_rows():
    """2^22 - 64 rows, of 256 columns: the last column's last row lies just below the descriptor's end. Rows of zeros
    but for the last 64, as above; the derivative rounded once to bf16, the gradient too."""
    from causal_tuner.kernels.loss import projection_loss
    rows, width, vocab = (1 << 22) - 64, 256, 130
    g = torch.Generator(device="cuda").manual_seed(1)
    hidden = torch.zeros(rows, width, device="cuda", dtype=BF16)
    hidden[-64:] = torch.randn(64, width, device="cuda", generator=g).to(BF16)
    head = (torch.randn(vocab, width, device="cuda", generator=g) * 0.1).to(BF16).requires_grad_()
    labels = torch.randint(vocab, (rows,), device="cuda", generator=g)
    run = lambda h, to: projection_loss(h, head, to, torch.ones(1, device="cuda").expand(len(h)), implementation="streamed",  # noqa: E731
                                        rows=slice(0, len(h)))
    dw, = torch.autograd.grad(run(hidden, labels), head)
    h = hidden[-64:].double()
    d = torch.softmax(h @ head.detach().double().T, -1)
    d[torch.arange(64), labels[-64:]] -= 1
    bound = (d.abs() * (2.0 ** -8 + 2.0 ** -16) + 2.0 ** -20).T @ h.abs()
    want = d.T @ h
    assert ((dw.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()
    with pytest.raises(ValueError, match="head's gradient"):
        run(hidden[:1].expand(rows + 1, width), labels[:1].expand(rows + 1))


def _repeated(count, tokens, g):
    """Row numbers with repeats, some outside the batch, and how often each row is given."""
    rows = torch.randint(tokens, (count,), device="cuda", generator=g)
    rows[::7] = -1 - rows[::7]
    rows[3::11] = tokens + (rows[3::11] << 33)
    inside = rows[(rows >= 0) & (rows < tokens)]
    times = torch.bincount(inside, minlength=tokens)
    return rows, times


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("count,tokens", [(2, 1), (40, 3), (130, 50), (900, 200), (1000, 100000)])
@pytest.mark.parametrize("teacher", [False, True])
def test_rows_given_twice_count_twice(teacher, count, tokens, dtype):
    """As once with their weight times that count: within the bounds of those rows, and the same bits on each call."""
    from causal_tuner.kernels.loss import distillation_loss, projection_loss
    g = torch.Generator(device="cuda").manual_seed(count)
    hidden = torch.randn(tokens, 72, device="cuda", generator=g).to(dtype).requires_grad_()
    head = (torch.randn(333, 72, device="cuda", generator=g) * 0.3).to(dtype).requires_grad_()
    weights = torch.rand(tokens, device="cuda", generator=g) + 0.1
    labels = torch.randint(333, (tokens, 3 if teacher else 1), device="cuda", generator=g)
    values = torch.randn(tokens, 3, device="cuda", generator=g)
    rows, times = _repeated(count, tokens, g)

    def run():
        if teacher:
            loss = distillation_loss(hidden, head, labels, values, weights, compute_dtype=dtype, rows=rows)
        else:
            loss = projection_loss(hidden, head, labels[:, 0], weights, implementation="streamed", compute_dtype=dtype, rows=rows)
        return (loss.detach(), *torch.autograd.grad(loss, (hidden, head)))
    got = run()
    chosen = times.nonzero().flatten()
    scaled = (weights * times)[chosen]
    want = reference(hidden[chosen], head, labels[chosen], values[chosen] if teacher else None, scaled)
    bound = bounds(want[3], scaled, dtype, dtype, dtype)
    # the head's gradient sums as many terms as there are rows given, not as there are rows
    more = count * 2.0 ** -24 * (want[3][8].abs().T @ hidden[chosen].detach().double().abs())
    check("loss", got[0], want[0], bound[0])
    check("dh", got[1][chosen], want[1], bound[1])
    check("dW", got[2], want[2], bound[2] + more)
    assert not got[1][times == 0].any()
    assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_captured_rows_that_change_between_replays():
    """The count of each row is taken anew by every replay."""
    from causal_tuner.kernels.loss import projection_loss
    g = torch.Generator(device="cuda").manual_seed(5)
    hidden = torch.randn(90, 64, device="cuda", generator=g).to(BF16).requires_grad_()
    head = (torch.randn(500, 64, device="cuda", generator=g) * 0.3).to(BF16)
    labels, weights = torch.randint(500, (90,), device="cuda", generator=g), torch.rand(90, device="cuda", generator=g) + 0.1
    rows = torch.arange(70, device="cuda")

    def step():
        loss = projection_loss(hidden, head, labels, weights, implementation="streamed", rows=rows)
        return (loss.detach(), *torch.autograd.grad(loss, (hidden,)))
    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        with torch.no_grad():
            rows.copy_(_repeated(70, 90, g)[0] if turn % 2 else torch.randperm(90, device="cuda", generator=g)[:70])
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


@pytest.mark.parametrize("frozen", [False, True])
def test_under_a_checkpoint(frozen):
    """The norm and the loss formed again in the backward: what is kept comes from the second forward."""
    from torch.utils.checkpoint import checkpoint

    from causal_tuner.kernels.loss import projection_loss
    from causal_tuner.modeling.norm import LayerNorm
    norm = LayerNorm(72, 1e-5, BF16, "cuda")
    x, head = _pitched(90, 72, 104, BF16, 1), _pitched(500, 72, 136, BF16, 2)
    head.requires_grad_(not frozen)
    labels, weights = torch.randint(500, (90,), device="cuda"), torch.rand(90, device="cuda") + 0.1
    rows = torch.tensor([3, 80, 3, 41], device="cuda")
    leaves = [x, norm.weight, norm.bias] + ([] if frozen else [head])
    step = lambda x, head: projection_loss(norm(x), head, labels, weights, implementation="streamed", rows=rows)  # noqa: E731
    want = torch.autograd.grad(step(x, head), leaves)
    got = torch.autograd.grad(checkpoint(step, x, head, use_reentrant=False), leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("h_type,w_type,compute", [(torch.float16, F32, BF16), (BF16, F32, F32), (F32, BF16, F32),
                                                   (torch.float16, BF16, F32), (torch.float64, F32, F32)])
def test_types_beside_the_computed_one(h_type, w_type, compute):
    """Operands of other types are brought to the computed one first; gradients come in their own."""
    from causal_tuner.kernels.loss import projection_loss
    g = torch.Generator(device="cuda").manual_seed(7)
    hidden = torch.randn(2, 35, 40, device="cuda", generator=g).to(compute).to(h_type).requires_grad_()
    head = (torch.randn(300, 40, device="cuda", generator=g) * 0.3).to(compute).to(w_type).requires_grad_()
    labels = torch.randint(300, (2, 35), device="cuda", generator=g, dtype=torch.int32)
    weights = torch.rand(2, 35, device="cuda", generator=g) + 0.1
    loss = projection_loss(hidden, head, labels, weights, implementation="streamed", compute_dtype=compute)
    dh, dw = torch.autograd.grad(loss, (hidden, head))
    assert dh.dtype == h_type and dw.dtype == w_type and dh.shape == hidden.shape
    h, w, flat = hidden.detach().reshape(-1, 40).to(compute), head.detach().to(compute), weights.flatten()
    want = reference(h, w, labels.reshape(-1, 1).long(), None, flat)
    bound = bounds(want[3], flat, compute, F32, F32)
    half = {torch.float16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24, torch.float64: 0.0}
    check("loss", loss.detach(), want[0], bound[0])
    # rounded to the leaf's type beside float32; float16's smallest step near zero is 2^-24
    for name, got, exact, b, t in (("dh", dh.reshape(-1, 40), want[1], bound[1], h_type), ("dW", dw, want[2], bound[2], w_type)):
        check(name, got, exact, b + half[t] * (exact.abs() + b) + (2.0 ** -25 if t == torch.float16 else 0.0))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_tokens(dtype):
    from causal_tuner.kernels.loss import distillation_loss, projection_loss
    hidden = torch.zeros(0, 40, device="cuda", dtype=dtype, requires_grad=True)
    head = torch.randn(30, 40, device="cuda").to(dtype).requires_grad_()
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    weights, entries = torch.zeros(0, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda")
    for loss in (projection_loss(hidden, head, none, weights, implementation="streamed", compute_dtype=dtype),
                 distillation_loss(hidden, head, entries, entries.float(), weights, compute_dtype=dtype)):
        dh, dw = torch.autograd.grad(loss, (hidden, head))
        assert loss.item() == 0 and dh.shape == hidden.shape and not dw.any()


def test_two_streams_at_once():
    """Calls of two streams share no scratch memory: both run together and give what each gives alone."""
    from causal_tuner.kernels.loss import projection_loss
    g = torch.Generator(device="cuda").manual_seed(3)
    cases = []
    for rows in (300, 41):
        hidden = torch.randn(rows, 256, device="cuda", generator=g).to(BF16).requires_grad_()
        head = (torch.randn(9000, 256, device="cuda", generator=g) * 0.1).to(BF16).requires_grad_()
        cases.append((hidden, head, torch.randint(9000, (rows,), device="cuda", generator=g),
                      torch.rand(rows, device="cuda", generator=g) + 0.1, torch.arange(rows, device="cuda") // 2))

    def step(hidden, head, labels, weights, rows):
        loss = projection_loss(hidden, head, labels, weights, implementation="streamed", rows=rows)
        return torch.autograd.grad(loss, (hidden, head))
    want = [step(*case) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(step(*case))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
