"""projection_loss(implementation="streamed") and distillation_loss (ct_head_loss_forward,
ct_head_loss_backward) against float64 from the definition, elementwise within bounds counted from
their roundings (head_loss_reference.py)."""

import math

import pytest
import torch

from head_loss_reference import bounds, check, reference

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _inputs(rows, width, vocab, dtype, seed=1, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    hidden = make(rows, width).to(dtype)
    head = (make(vocab, width) * scale / math.sqrt(width)).to(dtype)
    labels = torch.randint(vocab, (rows,), device="cuda", generator=g)
    weights = torch.rand(rows, device="cuda", generator=g) + 0.1
    return hidden.requires_grad_(), head.requires_grad_(), labels, weights


def _teacher(rows, vocab, entries, seed=2, holes=True):
    """Entries with equal indices, indices outside the vocabulary, values of -inf, NaN where there is
    no entry, and a row of none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    indices = torch.randint(vocab, (rows, entries), device="cuda", generator=g)
    values = torch.randn(rows, entries, device="cuda", generator=g) * 3
    if holes:
        gone = torch.rand(rows, entries, device="cuda", generator=g) < 0.2
        indices[gone] = torch.where(indices[gone] % 2 == 0, -1, vocab)
        values[gone] = math.nan
        values[torch.rand(rows, entries, device="cuda", generator=g) < 0.1] = -math.inf
        values[gone] = math.nan
        indices[rows // 2] = -1
    return indices, values


def _grads(loss, hidden, head, upstream=1.0):
    leaves = [t for t in (hidden, head) if t.requires_grad]
    return torch.autograd.grad(loss, leaves, torch.full_like(loss, upstream), retain_graph=True)


def _check(loss, hidden, head, indices, values, weights, dtype, temperature=1.0, normalizer=None, upstream=1.0):
    dh, dw = _grads(loss, hidden, head, upstream)
    want_loss, want_dh, want_dw, parts = reference(hidden.to(dtype), head.to(dtype), indices, values, weights, temperature,
                                                   normalizer, upstream)
    b_loss, b_dh, b_dw = bounds(parts, weights, dtype, hidden.dtype, head.dtype, temperature)
    check("loss", loss.detach(), want_loss, b_loss)
    check("dh", dh, want_dh, b_dh)
    check("dW", dw, want_dw, b_dw)
    return dh, dw


def _streamed(hidden, head, labels, weights, dtype, **kw):
    from causal_tuner.kernels.loss import projection_loss
    return projection_loss(hidden, head, labels, weights, implementation="streamed", compute_dtype=dtype, **kw)


SIZES = [(1, 64, 1), (1, 8, 2), (1, 512, 4099), (2, 72, 127), (17, 64, 128), (63, 200, 129), (64, 128, 1000),
         (65, 64, 255), (128, 136, 257), (129, 256, 513), (255, 64, 1025), (257, 512, 4099), (600, 320, 777),
         # wide rows and few entries: the logits' reduction in chunks
         (1, 4096, 300), (18, 2056, 328), (70, 1032, 129), (140, 2048, 500), (300, 1031, 1000), (700, 520, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_hard_labels(rows, width, vocab, dtype):
    hidden, head, labels, weights = _inputs(rows, width, vocab, dtype)
    _check(_streamed(hidden, head, labels, weights, dtype), hidden, head, labels[:, None], None, weights, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [1, 7, 91, 130])
def test_widths_that_fill_no_vector(width, dtype):
    hidden, head, labels, weights = _inputs(70, width, 1003, dtype)
    _check(_streamed(hidden, head, labels, weights, dtype), hidden, head, labels[:, None], None, weights, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("normalizer", [False, True])
@pytest.mark.parametrize("rows,width,vocab,entries,temperature", [
    (1, 64, 300, 1, 1.0), (3, 64, 17, 40, 2.0), (33, 72, 1000, 8, 0.5), (100, 128, 4099, 64, 2.0), (130, 64, 513, 65, 4.0),
    (300, 256, 2050, 128, 1.0), (20, 64, 5000, 1024, 1.0), (33, 1024, 700, 30, 2.0), (260, 777, 90, 100, 0.5)])
def test_teacher(rows, width, vocab, entries, temperature, normalizer, dtype):
    from causal_tuner.kernels.loss import distillation_loss
    hidden, head, _, weights = _inputs(rows, width, vocab, dtype)
    indices, values = _teacher(rows, vocab, entries, holes=entries > 1)
    norm = None
    if normalizer:
        norm = torch.logsumexp(values.masked_fill((indices < 0) | (indices >= vocab), -math.inf) / temperature, -1)
        norm = norm.clamp_min(-10) + 0.3
    loss = distillation_loss(hidden, head, indices, values, weights, temperature=temperature, log_normalizer=norm,
                             compute_dtype=dtype)
    dh, _ = _check(loss, hidden, head, indices, values, weights, dtype, temperature, norm, upstream=0.7)
    if entries > 1:
        assert not dh[rows // 2].any()


@pytest.mark.parametrize("teacher", [False, True])
def test_many_pieces(teacher):
    """More exponentials than one piece holds: running maxima and sums across pieces."""
    from causal_tuner.kernels.loss import distillation_loss
    rows, width, vocab = 4100, 64, 70001
    hidden, head, labels, weights = _inputs(rows, width, vocab, BF16)
    weights = weights / rows
    if teacher:
        indices, values = _teacher(rows, vocab, 16)
        loss = distillation_loss(hidden, head, indices, values, weights)
    else:
        indices, values = labels[:, None], None
        loss = _streamed(hidden, head, labels, weights, BF16)
    _check(loss, hidden, head, indices, values, weights, BF16)


@pytest.mark.parametrize("rows,width,vocab", [(513, 72, 14600), (600, 33, 13200), (1030, 264, 8200), (512, 72, 14600)])
def test_float32_on_wide_and_narrow_tiles(rows, width, vocab):
    """More tiles than the narrow one takes from 513 rows on, in terms that lie in memory; 512 rows beside it."""
    from causal_tuner.kernels.loss import distillation_loss
    hidden, head, labels, weights = _inputs(rows, width, vocab, F32)
    weights = weights / rows
    _check(_streamed(hidden, head, labels, weights, F32), hidden, head, labels[:, None], None, weights, F32)
    indices, values = _teacher(rows, vocab, 20)
    loss = distillation_loss(hidden, head, indices, values, weights, temperature=2.0, compute_dtype=F32)
    _check(loss, hidden, head, indices, values, weights, F32, 2.0)


@pytest.mark.parametrize("dtype,rows,vocab", [(BF16, 4100, 70001), (F32, 2100, 45001)])
@pytest.mark.parametrize("order", [1, -1])
def test_maxima_that_move_between_pieces(order, dtype, rows, vocab):
    """The sums of the pieces before are brought to a larger shift, or later units to theirs."""
    hidden, head, labels, weights = _inputs(rows, 64, vocab, dtype)
    with torch.no_grad():
        size = torch.linspace(0.2, 40.0, vocab, device="cuda")[:, None]
        head.mul_(size if order > 0 else size.flip(0))
    weights = weights / rows
    _check(_streamed(hidden, head, labels, weights, dtype), hidden, head, labels[:, None], None, weights, dtype)


def test_offsets_past_32_bits():
    """A head of 2.3e9 values, nearly all rows zero, so that what they add is known: logits of 0 and no
    gradient of the hidden rows."""
    vocab, width, rows = 140000, 16384, 3
    filled = torch.tensor([0, 1, vocab // 2, vocab - 2, vocab - 1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    hidden = torch.randn(rows, width, device="cuda", generator=g).to(BF16).requires_grad_()
    head = torch.zeros(vocab, width, device="cuda", dtype=BF16)
    head[filled] = (torch.randn(5, width, device="cuda", generator=g) * 0.1).to(BF16)
    head.requires_grad_()
    labels = torch.tensor([vocab - 1, 0, vocab - 2], device="cuda")
    weights = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    loss = _streamed(hidden, head, labels, weights, BF16)
    dh, dw = _grads(loss, hidden, head)
    h, w, c = hidden.detach().double(), head.detach()[filled].double(), weights.double()[:, None]
    logits = h @ w.T
    z = logits.exp().sum(-1, keepdim=True) + (vocab - 5)
    q = (filled == labels[:, None]).double()
    d = c * (logits.exp() / z - q)
    # logits are float32 chains of 16384 products: 2^-10 of a few dozen; the results are rounded to bf16
    assert abs(loss.item() - (c * (z.log() - (q * logits).sum(-1, keepdim=True))).sum().item()) < 0.05
    assert ((dh.double() - d @ w).norm(dim=-1) <= 2e-2 * (d @ w).norm(dim=-1)).all()
    want = d.T @ h
    assert ((dw[filled].double() - want).norm(dim=-1) <= 2e-2 * want.norm(dim=-1)).all()
    other = (c / z).T @ h   # of a row of zeros
    for row in (2, vocab // 2 + 1, vocab - 3):
        assert (dw[row].double() - other[0]).norm() <= 2e-2 * other.norm()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [1e-3, 40.0, 400.0])
def test_logits_of_any_size(scale, dtype):
    """Units whose maxima are far apart, above and below each other's shifts, in every order."""
    hidden, head, labels, weights = _inputs(140, 64, 1500, dtype, scale=scale)
    with torch.no_grad():
        head[300:600] *= 3
        head[900:1000] *= 0.01
    _check(_streamed(hidden, head, labels, weights, dtype), hidden, head, labels[:, None], None, weights, dtype)


def test_all_logits_far_below_and_above_zero():
    """A common offset of the logits, of either sign, leaves the probabilities."""
    for offset in (-300.0, -47.0, 49.0, 300.0):
        hidden, head, labels, weights = _inputs(70, 72, 700, BF16)
        with torch.no_grad():
            hidden[:, -1], head[:, -1] = 1.0, offset
        _check(_streamed(hidden, head, labels, weights, BF16), hidden, head, labels[:, None], None, weights, BF16)


def test_confident_rows_keep_their_gradient():
    """Labels of probability near one: 1 - p is not the difference of two roundings."""
    hidden, head, labels, weights = _inputs(80, 128, 900, BF16)
    with torch.no_grad():
        head.mul_(0.2)
        hidden.copy_((head[labels].float() * 180 + hidden.float() * 0.05).to(BF16))
    loss = _streamed(hidden, head, labels, weights, BF16)
    p = torch.softmax(hidden.double() @ head.double().T, -1).gather(1, labels[:, None])
    assert (p > 0.99).float().mean() > 0.5
    dh, dw = _check(loss, hidden, head, labels[:, None], None, weights, BF16)
    want = reference(hidden, head, labels[:, None], None, weights)[1]
    assert ((dh.double() - want).norm(dim=-1) <= 0.02 * want.norm(dim=-1)).all()


def test_labels_outside_the_vocabulary_leave_log_z():
    """As weighted_ce: the target's term is 0."""
    hidden, head, labels, weights = _inputs(5, 64, 100, BF16)
    labels[1], labels[3] = -100, 100
    _check(_streamed(hidden, head, labels, weights, BF16), hidden, head, labels[:, None], None, weights, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [slice(3, 90), "indices", "weights", slice(5, 5)])
def test_row_selections(rows, dtype):
    """Rows outside the selection: no loss, a zero gradient, and what they hold does not matter."""
    from causal_tuner.kernels.loss import active_rows
    hidden, head, labels, weights = _inputs(100, 72, 333, dtype)
    chosen = torch.randperm(100, device="cuda")[:37] if rows in ("indices", "weights") else torch.arange(100, device="cuda")[rows]
    off = torch.ones(100, dtype=torch.bool, device="cuda")
    off[chosen] = False
    if rows == "weights":
        weights[off] = 0
        given = None
        assert not isinstance(active_rows(weights), slice)
    else:
        given = chosen if rows == "indices" else rows
    with torch.no_grad():
        hidden[off] = math.nan
        labels[off] = -5
    loss = _streamed(hidden, head, labels, weights, dtype, rows=given)
    dh, dw = _grads(loss, hidden, head)
    assert not dh[off].any()
    part = hidden.detach()[chosen].requires_grad_()
    want_loss, want_dh, want_dw, parts = reference(part, head, labels[chosen][:, None], None, weights[chosen])
    b = bounds(parts, weights[chosen], dtype, dtype, dtype)
    for name, got, want, bound in (("loss", loss.detach(), want_loss, b[0]), ("dh", dh[chosen], want_dh, b[1]),
                                   ("dW", dw, want_dw, b[2])):
        check(name, got, want, bound + 1e-30)


def test_rows_outside_the_batch_have_no_loss():
    hidden, head, labels, weights = _inputs(40, 64, 200, BF16)
    rows = torch.tensor([3, 40, 7, -1, 1 << 40, 20], device="cuda")
    kept = torch.tensor([3, 7, 20], device="cuda")
    got = _streamed(hidden, head, labels, weights, BF16, rows=rows)
    want = _streamed(hidden, head, labels, weights, BF16, rows=kept)
    assert torch.equal(got, want)
    for a, b in zip(_grads(got, hidden, head), _grads(want, hidden, head)):
        assert torch.equal(a, b) or torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=1e-6)


@pytest.mark.parametrize("rows", [50, 300])
def test_float32_parameters_computed_in_bf16(rows):
    """A float32 head and hidden states: operands rounded to bf16, gradients in float32."""
    hidden, head, labels, weights = _inputs(rows, 128, 1100, F32)
    with torch.no_grad():   # values that bf16 holds, so that the cast loses nothing
        hidden.copy_(hidden.to(BF16))
        head.copy_(head.to(BF16))
    dh, dw = _check(_streamed(hidden, head, labels, weights, BF16), hidden, head, labels[:, None], None, weights, BF16)
    assert dh.dtype == dw.dtype == F32


def test_strides_and_alignments():
    base_h, base_w, labels, weights = _inputs(90, 136, 700, BF16)
    with torch.no_grad():
        wide_h = torch.randn(90, 2, 150, device="cuda").to(BF16)
        wide_w = torch.randn(700, 141, device="cuda").to(BF16)
        wide_h[:, 1, 3:139], wide_w[:, 5:] = base_h, base_w
        column = base_w.detach().T.contiguous().T
        far_h, far_w = (torch.empty(n, 1 << 20 | 8, device="cuda", dtype=BF16)[:, 8:144] for n in (90, 700))
        far_h.copy_(base_h)
        far_w.copy_(base_w)
    views = [(far_h, far_w), (wide_h.detach()[:, 1, 3:139], wide_w.detach()[:, 5:]), (base_h.detach()[:, :], column),
             (base_h.detach().T.contiguous().T, base_w.detach())]
    loss = _streamed(base_h, base_w, labels, weights, BF16)
    want = (loss.detach(), *_grads(loss, base_h, base_w))
    for h, w in views:
        h, w = h.requires_grad_(), w.requires_grad_()
        loss = _streamed(h, w, labels, weights, BF16)
        got = (loss.detach(), *_grads(loss, h, w))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("frozen", ["head", "hidden"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_side_frozen(frozen, dtype):
    hidden, head, labels, weights = _inputs(150, 128, 900, dtype)
    both = _grads(_streamed(hidden, head, labels, weights, dtype), hidden, head)
    hidden.requires_grad_(frozen != "hidden")
    head.requires_grad_(frozen != "head")
    one, = _grads(_streamed(hidden, head, labels, weights, dtype), hidden, head)
    assert torch.equal(one, both[0] if frozen == "head" else both[1])
    with torch.no_grad():
        alone = _streamed(hidden, head, labels, weights, dtype)
    assert not alone.requires_grad
    assert torch.allclose(alone, _streamed(hidden, head, labels, weights, dtype).detach(), rtol=1e-6)


def test_backward_repeats_and_scales():
    hidden, head, labels, weights = _inputs(200, 64, 3000, BF16)
    loss = _streamed(hidden, head, labels, weights, BF16)
    first, second = _grads(loss, hidden, head), _grads(loss, hidden, head)
    four = _grads(loss, hidden, head, 4.0)
    for a, b, c in zip(first, second, four):
        assert torch.equal(a, b) and torch.equal(4 * a, c)
    again = _streamed(hidden, head, labels, weights, BF16)
    assert torch.equal(loss, again)
    for a, b in zip(first, _grads(again, hidden, head)):
        assert torch.equal(a, b)


def test_gradient_against_differences():
    hidden, head, labels, weights = _inputs(6, 8, 40, F32)
    indices, values = _teacher(6, 40, 4)
    from causal_tuner.kernels.loss import distillation_loss
    run = lambda: distillation_loss(hidden, head, indices, values, weights, temperature=2.0, compute_dtype=F32)  # noqa: E731
    dh, dw = _grads(run(), hidden, head)
    step = 2.0 ** -6
    for tensor, grad, places in ((hidden, dh, [(0, 0), (1, 5), (5, 7)]), (head, dw, [(0, 1), (7, 3), (39, 7)])):
        for at in places:
            with torch.no_grad():
                old = tensor[at].item()
                tensor[at] = old + step
                up = run().item()
                tensor[at] = old - step
                down = run().item()
                tensor[at] = old
            # two losses of size ~10 rounded to float32 (2^-20), and the third derivative times step^2 / 6
            assert abs((up - down) / (2 * step) - grad[at].item()) < 2 * 10 * 2.0 ** -23 / step + step ** 2 * 5


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_not_finite_stays_in_its_row(dtype):
    hidden, head, labels, weights = _inputs(70, 64, 300, dtype)
    head.requires_grad_(False)
    with torch.no_grad():
        hidden[5, 3] = math.nan
        hidden[9, 0] = math.inf
    loss = _streamed(hidden, head, labels, weights, dtype)
    dh, = _grads(loss, hidden, head)
    assert torch.isnan(loss) and torch.isnan(dh[5]).any() and torch.isnan(dh[9]).any()
    rest = torch.ones(70, dtype=torch.bool)
    rest[[5, 9]] = False
    want = reference(hidden.detach()[rest], head, labels[rest][:, None], None, weights[rest])
    check("dh", dh[rest], want[1], bounds(want[3], weights[rest], dtype, dtype, dtype)[1])


def test_other_stream_and_captured_replays():
    """Forward and backward in one graph beside eager calls, two graphs, new inputs each replay."""
    from causal_tuner.kernels.loss import distillation_loss
    hidden, head, labels, weights = _inputs(150, 128, 2000, BF16)
    indices, values = _teacher(150, 2000, 8)
    rows = slice(0, 150)

    def step():
        loss = distillation_loss(hidden, head, indices, values, weights, rows=rows) \
            + _streamed(hidden, head, labels, weights, BF16, rows=rows)
        return (loss.detach(), *torch.autograd.grad(loss, (hidden, head)))
    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for turn in range(3):
        with torch.no_grad():
            hidden.copy_(torch.randn_like(hidden))
        want = step()
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_statistics_alone_in_pieces():
    """Without gradients: so many rows that the units' statistics come to more than one piece, against
    the same rows in parts. A unit's sum is the same in both; joining 71 of them in two orders differs
    by at most 2 x 71 x 2^-24 < 2^-16 of Z, of the losses' mean (log 9000 and more) by less than 2^-19,
    and the nine losses are rounded by 2^-24 each."""
    rows, width, vocab = 1 << 20, 64, 9000   # 71 units of 8 bytes a row
    hidden, head, labels, weights = _inputs(rows, width, vocab, BF16)
    with torch.no_grad():
        weights = weights.abs() / rows
        whole = _streamed(hidden, head, labels, weights, BF16).double()
        step = rows // 8
        parts = sum(_streamed(hidden, head, labels, weights, BF16, rows=slice(i, i + step)).double()
                    for i in range(0, rows, step))
    assert abs(whole - parts) <= (2.0 ** -19 + 2.0 ** -22) * parts.abs()


def test_refusals():
    from causal_tuner.kernels.loss import distillation_loss
    hidden, head, labels, weights = _inputs(4, 16, 30, BF16)
    with pytest.raises(NotImplementedError):
        _streamed(hidden, head, labels, weights, torch.float16)
    with pytest.raises(ValueError, match="cpu"):
        _streamed(hidden, head.detach().cpu(), labels, weights, BF16)
    with pytest.raises(ValueError, match="targets"):
        _streamed(hidden, head, labels.cpu(), weights, BF16)
    with pytest.raises(ValueError, match="indices"):
        distillation_loss(hidden, head, labels[:, None].cpu(), torch.zeros(4, 1), weights)
    with pytest.raises(ValueError, match="at once"):
        tall = torch.zeros(1, 16, device="cuda", dtype=BF16).expand(1 << 24, 16)
        _streamed(tall, head, labels[:1].expand(1 << 24), weights[:1].expand(1 << 24), BF16, rows=slice(0, 1 << 24))
    with pytest.raises(ValueError, match="width"):
        _streamed(hidden.new_zeros(4, 65544), hidden.new_zeros(2, 65544), labels, weights, BF16)
    for rows in (torch.ones(4, dtype=torch.bool, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda"),
                 slice(0, 4, 2)):
        with pytest.raises(ValueError, match="rows"):
            _streamed(hidden, head, labels, weights, BF16, rows=rows)
    loss = _streamed(hidden, head, labels, weights, BF16)
    grad, = torch.autograd.grad(loss, hidden, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
