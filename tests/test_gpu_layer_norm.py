"""layer_norm (ct_layer_norm_forward, ct_layer_norm_backward) against float64 from the definition,
elementwise within bounds counted from its roundings (`_check`)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: UNIT}
EPS = 1e-5


def _inputs(rows, width, dtype, kept, bias=True, mean=0.7, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = (make(rows, width) * torch.exp(0.5 * make(width)) + mean * make(rows, 1)).to(dtype).requires_grad_()
    weight = (1 + 0.2 * make(width)).to(kept).requires_grad_()
    b = (0.1 * make(width)).to(kept).requires_grad_() if bias else None
    return x, weight, b, make(rows, width).to(dtype)


def _check(x, weight, bias, dy, got, eps=EPS):
    """The mean is a float32 sum of `width` terms (in runs of at most 16 and a tree: width / 64 + 16
    roundings of the sum of magnitudes), so x - mean is off by that and its own rounding; rstd by half the
    variance's relative error, which is of the same size, and the kernel's square root and division
    (4 units together); every further product and sum rounds once; the result once to its type."""
    leaves = [None if t is None else t.detach().double().requires_grad_() for t in (x, weight, bias)]
    x64, w64, b64 = leaves
    width = x.shape[-1]
    terms = (width / 64 + 32) * UNIT
    mean = x64.mean(-1, keepdim=True)
    c = x64 - mean
    var = c.square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    n = c * rstd
    w = torch.ones_like(mean[0]) if w64 is None else w64
    y = n * w + (0 if b64 is None else b64)
    want = [y] + list(torch.autograd.grad(y, [t for t in leaves if t is not None], dy.double()))
    x64, mean, c, rstd, n, w = (t.detach() for t in (x64, mean, c, rstd, n, w))
    off_mean = terms * x64.abs().mean(-1, keepdim=True)
    off_c = off_mean + UNIT * (c.abs() + mean.abs())
    # c enters the variance linearly with a zero sum: a common offset only by its square
    off_rstd = rstd * (terms + 6 * UNIT + (rstd * off_mean).square() + 2 * UNIT * (rstd * (c.abs() + mean.abs())).amax(-1, keepdim=True))
    off_n = rstd * off_c + c.abs() * off_rstd + 2 * UNIT * n.abs()
    off_y = off_n * w.abs() + 3 * UNIT * (n * w).abs() + 2 * UNIT * y.detach().abs()
    d = dy.double()
    g = d * w
    g_sum, gn_sum = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    off_a, off_b = terms * g_sum, terms * gn_sum + (g.abs() * off_n).mean(-1, keepdim=True)
    b = (g * n).mean(-1, keepdim=True).abs()
    inner = g.abs() + g_sum + (n * b).abs()
    off_dx = rstd * (4 * UNIT * inner + off_a + off_n * b + n.abs() * off_b) + off_rstd * inner
    rows = d.reshape(-1, width)
    sums = len(rows) * UNIT
    flat = lambda t: t.expand_as(d).reshape(-1, width)  # noqa: E731
    off_dw = (rows.abs() * (flat(off_n) + (sums + 2 * UNIT) * flat(n).abs())).sum(0)
    off_db = sums * rows.abs().sum(0)
    offs = [off_y, off_dx] + ([] if weight is None else [off_dw]) + ([] if bias is None else [off_db])
    for name, a, e, off in zip(("y", "dx", "dw", "db"), got, want, offs):
        e = e.detach()
        bound = off + HALF[a.dtype] * (e.abs() + off) + torch.finfo(a.dtype).smallest_normal * HALF[a.dtype] + 1e-30
        assert torch.isfinite(a).all(), name
        worst = ((a.double() - e).abs() / bound).max().item()
        assert worst <= 1, f"{name}: {worst:.3g} times its bound"


def _run(x, weight, bias, dy, eps=EPS):
    from causal_tuner.modeling.norm import layer_norm
    y = layer_norm(x, weight, bias, eps)
    with torch.no_grad():
        torch.testing.assert_close(layer_norm(x, weight, bias, eps), y.detach(), rtol=0, atol=0, equal_nan=True)
    leaves = [t for t in (x, weight, bias) if t is not None]
    return (y.detach(), *torch.autograd.grad(y, leaves, dy, retain_graph=True))


WIDTHS = [1, 2, 3, 8, 63, 64, 65, 255, 512, 513, 1000, 1023, 1024, 1032, 2048, 2056, 4096, 4097, 4104, 6144, 8192, 8200,
          10240, 16384, 16385, 16392, 33000, 65536, 70000]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, dtype):
    x, weight, bias, dy = _inputs(5, width, dtype, dtype)
    if width == 1:   # a row of one value has no spread: y = bias, and only bias has a gradient
        y, dx, dw, db = _run(x, weight, bias, dy)
        assert torch.equal(y[0], bias) and not dx.any() and not dw.any()
        return
    _check(x, weight, bias, dy, _run(x, weight, bias, dy))


@pytest.mark.parametrize("kept", [BF16, F16, F32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bias", [False, True])
def test_types(dtype, kept, bias):
    for width in (320, 77):
        x, weight, b, dy = _inputs(37, width, dtype, kept, bias)
        _check(x, weight, b, dy, _run(x, weight, b, dy))


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 511, 512, 513, 1025, 4099])
@pytest.mark.parametrize("width", [128, 1032, 2560])
def test_rows(rows, width):
    x, weight, bias, dy = _inputs(rows, width, BF16, F32)
    _check(x, weight, bias, dy, _run(x, weight, bias, dy))


def test_no_weight_no_bias_and_different_types():
    x, weight, bias, dy = _inputs(30, 96, BF16, BF16)
    _check(x, None, None, dy, _run(x, None, None, dy))
    _check(x, None, bias, dy, _run(x, None, bias, dy))
    wide = bias.detach().float() * 1.001
    got = _run(x, weight, wide.requires_grad_(), dy)
    assert got[2].dtype == BF16 and got[3].dtype == F32
    _check(x, weight, wide, dy, got)


def test_rows_with_a_large_mean():
    """The variance is of the differences from the mean, not of the squares."""
    for dtype in (F32, BF16):
        x, weight, bias, dy = _inputs(20, 1000, dtype, F32, mean=300.0)
        _check(x, weight, bias, dy, _run(x, weight, bias, dy))


def test_constant_and_zero_rows():
    x, weight, bias, dy = _inputs(4, 256, F32, F32)
    with torch.no_grad():
        x[0], x[2] = 0.0, 2.0
    y, dx, dw, db = _run(x, weight, bias, dy)
    assert torch.equal(y[0], bias) and torch.equal(y[2], bias)
    _check(x, weight, bias, dy, (y, dx, dw, db))


def test_no_rows():
    x, weight, bias, dy = _inputs(0, 64, BF16, BF16)
    y, dx, dw, db = _run(x, weight, bias, dy)
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


def test_shapes_strides_and_alignment():
    x, weight, bias, dy = _inputs(24, 80, BF16, BF16)
    want = _run(x, weight, bias, dy)
    big = torch.zeros(2, 12, 2, 81, device="cuda", dtype=BF16)
    big[:, :, 1, 1:] = x.detach().reshape(2, 12, 80)
    view = big[:, :, 1, 1:].requires_grad_()
    off = torch.empty(81, device="cuda", dtype=BF16)
    off[1:] = weight.detach()
    grads = torch.randn(2, 80, 12, device="cuda").to(BF16).transpose(1, 2)
    grads = grads.copy_(dy.reshape(2, 12, 80))
    got = _run(view, off[1:].requires_grad_(), bias, grads)
    _check(x, weight, bias, dy, [t.reshape(24, 80) if t.dim() == 3 else t for t in got])
    assert torch.equal(got[0].reshape(24, 80), want[0])


def test_some_gradients_only():
    x, weight, bias, dy = _inputs(33, 200, BF16, F32)
    full = _run(x, weight, bias, dy)
    from causal_tuner.modeling.norm import layer_norm
    for i, leaf in enumerate((x, weight, bias)):
        for other in (x, weight, bias):
            other.requires_grad_(other is leaf)
        grad, = torch.autograd.grad(layer_norm(x, weight, bias, EPS), leaf, dy)
        assert torch.equal(grad, full[i + 1])


def test_what_is_not_finite_stays_in_its_row():
    x, weight, bias, dy = _inputs(9, 128, BF16, BF16)
    with torch.no_grad():
        x[4, 7] = float("nan")
    y, dx, dw, db = _run(x, weight, bias, dy)
    rest = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.isnan(y[4]).all() and torch.isfinite(y[rest]).all() and torch.isfinite(dx[rest]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()


def test_repeats_other_stream_and_captured_replays():
    x, weight, bias, dy = _inputs(700, 1032, BF16, F32)
    want = _run(x, weight, bias, dy)
    assert all(torch.equal(a, b) for a, b in zip(want, _run(x, weight, bias, dy)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(x, weight, bias, dy)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    from causal_tuner.modeling.norm import layer_norm

    def step():
        y = layer_norm(x, weight, bias, EPS)
        return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), dy))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for turn in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        want = step()
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_module_and_gradient_against_differences():
    from causal_tuner.modeling.norm import LayerNorm
    norm = LayerNorm(48, EPS, F32, "cuda")
    assert LayerNorm(48, EPS, BF16, "cuda", bias=False).bias is None
    x, _, _, dy = _inputs(3, 48, F32, F32)
    grads = torch.autograd.grad(norm(x), (x, norm.weight, norm.bias), dy)
    run = lambda: (norm(x).double() * dy.double()).sum().item()  # noqa: E731
    step = 2.0 ** -7
    for tensor, grad, at in ((x, grads[0], (1, 5)), (norm.weight, grads[1], (7,)), (norm.bias, grads[2], (47,))):
        with torch.no_grad():
            old = tensor[at].item()
            tensor[at] = old + step
            up = run()
            tensor[at] = old - step
            down = run()
            tensor[at] = old
        # 48 values of y rounded to 2^-24 of about 3, over two steps; third derivatives of order one
        assert abs((up - down) / (2 * step) - grad[at].item()) < 48 * 3 * UNIT * 4 / step + 2 * step ** 2


def test_more_rows_than_one_launch_holds():
    """2^26 + 5 rows, whose statistics and values are those that the rows have by themselves."""
    from causal_tuner.modeling.norm import layer_norm
    rows, width = (1 << 26) + 5, 8
    x = torch.randn(1 << 20, width, device="cuda", dtype=BF16).repeat(65, 1)[:rows].requires_grad_()
    weight, bias = torch.randn(2, width, device="cuda")
    y = layer_norm(x, weight, bias)
    dy = y.detach().roll(1, -1)
    dx, = torch.autograd.grad(y, x, dy)
    for first in (0, (1 << 21) - 3, (1 << 25) - 1, (1 << 26) - 2, rows - 7):
        part = x.detach()[first:first + 7].clone().requires_grad_()
        want = layer_norm(part, weight, bias)
        assert torch.equal(y[first:first + 7], want), first
        assert torch.equal(dx[first:first + 7], torch.autograd.grad(want, part, dy[first:first + 7])[0]), first


def test_refusals():
    from causal_tuner.modeling.norm import layer_norm
    x, weight, bias, dy = _inputs(4, 16, F32, F32)
    with pytest.raises(NotImplementedError):
        layer_norm(x.double(), weight, bias)
    with pytest.raises(ValueError, match="cpu"):
        layer_norm(x, weight.detach().cpu(), bias)
    y = layer_norm(x, weight, bias)
    grad, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
