"""orthogonalize and FusedMuon (ct_muon) against the iteration in float64.

Bounds. The steps run in double, so what is left is the float32 product of the final r x r
matrix Q (rounded once, e = 2^-24) with M / |M|: (r + 4) e |Q| |M| / |M|_F, doubled for second
order and the double steps, and half a step u of the result's type. In a step, M itself is a
float32 combination: three roundings, which the iteration (slope at most a^steps) carries to
3 e a^steps in norm; the update and the parameter are rounded in float32 and stored in their type."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
E32 = 2.0 ** -24


def _reference(m, steps=5, eps=1e-7, coefficients=(A, B, C)):
    """(X_steps, elementwise bound before the output's own rounding) in float64."""
    a, b, c = coefficients
    x = m.double()
    wide = x.T if x.shape[0] > x.shape[1] else x
    x0 = wide / wide.norm().clamp(min=eps)
    x, q = x0, torch.eye(len(x0), dtype=torch.float64, device=m.device)
    for _ in range(steps):
        g = x @ x.T
        p = a * torch.eye(len(x0), dtype=torch.float64, device=m.device) + b * g + c * (g @ g)
        x, q = p @ x, p @ q
    bound = 2 * (len(x0) + 4) * E32 * (q.abs() @ x0.abs())
    return (x.T, bound.T) if m.shape[0] > m.shape[1] else (x, bound)


def _check(got, m, **kw):
    want, bound = _reference(m, **kw)
    u = torch.finfo(m.dtype).eps / 2
    assert got.shape == m.shape and got.dtype == m.dtype and torch.isfinite(got).all()
    over = (got.double() - want).abs() - bound - u * (want.abs() + bound) - 1e-37
    assert over.max() <= 0, f"{tuple(m.shape)} {m.dtype}: {over.max()} over a bound of {bound.max()}"


def _matrix(shape, dtype, decades=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g, dtype=torch.float64)
    if decades is not None:
        u, _, v = torch.linalg.svd(x, full_matrices=False)
        x = (u * torch.logspace(0, -decades, min(shape), dtype=torch.float64)) @ v
    return (x * 1e-3).to("cuda", dtype)


SHAPES = [(1, 1), (1, 7), (5, 1), (3, 3), (16, 1024), (1024, 16), (31, 33), (33, 31), (64, 64), (65, 200), (130, 1111),
          (2049, 64), (100, 300), (300, 100), (40, 516), (516, 252), (160, 640), (255, 257), (256, 4096), (4100, 128), (8, 3001), (300, 513), (700, 290)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype):
    from causal_tuner.optim import orthogonalize
    m = _matrix(shape, dtype)
    kept = m.clone()
    _check(orthogonalize(m), m)
    assert torch.equal(m, kept)


@pytest.mark.parametrize("decades", [1, 2, 3, 5])
def test_spectra_over_decades(decades):
    from causal_tuner.optim import orthogonalize
    m = _matrix((96, 500), torch.float32, decades)
    _check(orthogonalize(m), m)


def test_many_matrices_of_mixed_kinds_in_one_call():
    from causal_tuner.optim import orthogonalize
    inputs = [_matrix(s, t, seed=i) for i, (s, t) in enumerate(
        [((16, 100), torch.float32), ((100, 16), torch.bfloat16), ((70, 70), torch.float32), ((0, 5), torch.float32),
         ((256, 300), torch.bfloat16)] * 12)]
    strided = _matrix((64, 90), torch.float32).T
    inputs.append(strided)
    results = orthogonalize(inputs)
    assert len(results) == len(inputs)
    for got, m in zip(results, inputs):
        if m.numel():
            _check(got, m)
        assert got.shape == m.shape
    again = orthogonalize(inputs)
    assert all(torch.equal(x, y) for x, y in zip(results, again))


def test_zero_tiny_and_infinite_matrices():
    from causal_tuner.optim import orthogonalize
    zero, tiny = torch.zeros(20, 30, device="cuda"), _matrix((20, 30), torch.float32) * 1e-6
    bad = _matrix((20, 30), torch.float32)
    bad[3, 4] = float("inf")
    x, y, z = orthogonalize([zero, tiny, bad])
    assert not x.any()
    _check(y, tiny)
    assert torch.isnan(z).all()


def test_more_matrices_than_workgroups():
    """Workgroups of the last product go from one matrix to the next, of other sizes, kinds and
    alignments."""
    from causal_tuner.optim import orthogonalize
    sizes = [(8, 20), (100, 36), (5, 7), (40, 516), (1, 1), (260, 270), (33, 31), (1030, 24), (70, 200)]
    matrices = [_matrix(sizes[i % len(sizes)], torch.float32, seed=i) for i in range(330)]
    matrices[1::11] = [m.new_empty(m.numel() + 1)[1:].view(m.shape).copy_(m) for m in matrices[1::11]]
    for m, got in zip(matrices, orthogonalize(matrices)):
        _check(got, m)


@pytest.mark.parametrize("steps,coefficients", [(1, (2.0, -1.5, 0.5)), (2, (A, B, C)), (3, (1.875, -1.25, 0.375)),
                                                (8, (A, B, C))])
def test_steps_and_coefficients(steps, coefficients):
    from causal_tuner.optim import orthogonalize
    m = _matrix((40, 100), torch.float32)
    _check(orthogonalize(m, steps=steps, coefficients=coefficients), m, steps=steps, coefficients=coefficients)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
def test_muon_steps(dtype, nesterov, adjust):
    from causal_tuner.optim import FusedMuon
    shapes = [(16, 256), (256, 16), (128, 300), (40, 40)]
    params = [torch.nn.Parameter(_matrix(s, dtype, seed=i) * 20) for i, s in enumerate(shapes)]
    skipped = torch.nn.Parameter(_matrix((4, 4), dtype))
    lr, decay, mu = 0.02, 0.1, 0.9
    optimizer = FusedMuon([*params, skipped], lr=lr, weight_decay=decay, momentum=mu, nesterov=nesterov,
                          adjust_lr_fn=adjust)
    unchanged = skipped.detach().clone()
    momentum = [torch.zeros(s, dtype=torch.float64, device="cuda") for s in shapes]
    u = torch.finfo(dtype).eps / 2
    for step in range(3):
        before = [p.detach().double() for p in params]
        for i, p in enumerate(params):
            p.grad = _matrix(shapes[i], dtype, seed=100 * step + i)
        optimizer.step()
        for p, old, m in zip(params, before, momentum):
            buffer = optimizer.state[p]["momentum_buffer"]
            m.mul_(mu).add_(p.grad.double(), alpha=1 - mu)
            assert buffer.dtype == torch.float32
            assert ((buffer.double() - m).abs() <= 4 * (step + 1) * E32 * (m.abs() + p.grad.abs().max())).all()
            m.copy_(buffer)   # from here on with what the optimizer holds
            direction, bound = _reference(mu * m + (1 - mu) * p.grad.double() if nesterov else m)
            rows, cols = p.shape
            factor = lr * (0.2 * max(rows, cols) ** 0.5 if adjust else max(1.0, rows / cols) ** 0.5)
            want = old * (1 - lr * decay) - factor * direction
            allowed = factor * (bound + 3 * E32 * A ** 5 + 4 * E32 * direction.abs()) + 4 * E32 * old.abs()
            over = (p.double() - want).abs() - allowed - u * (want.abs() + allowed)
            assert over.max() <= 0, f"{tuple(p.shape)}: {over.max()} over"
    assert torch.equal(skipped, unchanged) and "momentum_buffer" not in optimizer.state[skipped]


def test_muon_against_torch_and_its_state():
    """torch.optim.Muon runs its steps in bfloat16: parameters agree to that (each step's update
    within 2^-8 a few times over its norm), momenta to float32."""
    from causal_tuner.optim import FusedMuon
    start = [_matrix(s, torch.float32, seed=i) for i, s in enumerate([(32, 200), (200, 32)])]
    ours, theirs = ([torch.nn.Parameter(m.clone()) for m in start] for _ in range(2))
    a, b = FusedMuon(ours, lr=0.02), torch.optim.Muon(theirs, lr=0.02)
    for step in range(2):
        for x, y in zip(ours, theirs):
            x.grad = _matrix(tuple(x.shape), torch.float32, seed=step + 7)
            y.grad = x.grad.clone()
        a.step()
        b.step()
    for x, y, m in zip(ours, theirs, start):
        moved = (y - m).norm()
        assert (x - y).norm() <= 0.05 * moved
        torch.testing.assert_close(a.state[x]["momentum_buffer"], b.state[y]["momentum_buffer"], rtol=1e-6, atol=1e-9)
    fresh = FusedMuon([torch.nn.Parameter(m.clone().bfloat16()) for m in start])
    fresh.load_state_dict(copy.deepcopy(b.state_dict()))
    for p, y in zip(fresh.param_groups[0]["params"], theirs):
        assert fresh.state[p]["momentum_buffer"].dtype == torch.float32
        assert torch.equal(fresh.state[p]["momentum_buffer"], b.state[y]["momentum_buffer"])
        p.grad = torch.ones_like(p)
    fresh.step()
    assert fresh.param_groups[0]["lr"] == 0.02


def test_captured_steps_replay():
    """orthogonalize and a step in a graph, replayed with new gradients between eager work; the
    plan of unseen shapes is refused inside a capture."""
    from causal_tuner.optim import FusedMuon, orthogonalize
    shapes = [(24, 200), (200, 24), (100, 300)]
    params, twins = ([torch.nn.Parameter(_matrix(s, torch.float32, seed=i)) for i, s in enumerate(shapes)]
                     for _ in range(2))
    a, b = FusedMuon(params, lr=0.01), FusedMuon(twins, lr=0.01)
    for p, t in zip(params, twins):
        p.grad, t.grad = torch.zeros_like(p), torch.zeros_like(t)
    a.step()   # buffers and plan exist; zero gradients leave only the decay
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
        made = orthogonalize([p.grad for p in params])
    for seed in range(3):
        for i, (p, t) in enumerate(zip(params, twins)):
            p.grad.copy_(_matrix(shapes[i], torch.float32, seed=50 + 3 * seed + i))
            t.grad.copy_(p.grad)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, t) for p, t in zip(params, twins))
        assert all(torch.equal(x, y) for x, y in zip(made, orthogonalize([t.grad for t in twins])))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            orthogonalize(torch.ones(11, 13, device="cuda"))
    torch.cuda.synchronize()
    fresh = torch.nn.Parameter(params[0].detach().clone())   # of a known shape, but without a buffer
    fresh.grad = torch.ones_like(fresh)
    orthogonalize(fresh.grad)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            FusedMuon([fresh]).step()
    torch.cuda.synchronize()
    _check(orthogonalize(params[0].detach()), params[0].detach())


def test_other_streams_and_unaligned_storage():
    from causal_tuner.optim import orthogonalize
    inputs = [_matrix((64, 301), torch.float32), _matrix((300, 130), torch.bfloat16)]
    shifted = []
    for m in inputs:   # contiguous, but no 16-byte start
        buffer = torch.empty(m.numel() + 1, device="cuda", dtype=m.dtype)
        shifted.append(buffer[1:].view(m.shape).copy_(m))
    torch.cuda.synchronize()
    results = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            results.append(orthogonalize(shifted))
    torch.cuda.synchronize()
    for result in results:
        for got, m in zip(result, inputs):
            _check(got, m)


def test_device_refusals():
    from causal_tuner.optim import FusedMuon, orthogonalize
    with pytest.raises(NotImplementedError):
        orthogonalize(torch.zeros(3, 3, device="cuda", dtype=torch.float16))
    p = torch.nn.Parameter(torch.zeros(6, 4, device="cuda"))
    p.grad = torch.zeros(4, 6, device="cuda").T
    with pytest.raises(NotImplementedError, match="contiguous"):
        FusedMuon([p]).step()
    p.grad = torch.zeros(6, 4, device="cuda")
    optimizer = FusedMuon([p])
    optimizer.state[p]["momentum_buffer"] = torch.zeros(6, 4, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="momentum_buffer"):
        optimizer.step()


def _low_rank(shape, rank, dtype, seed=0):
    """(matrix of whole numbers, exact in `dtype`; its factors in float64)."""
    g = torch.Generator().manual_seed(seed)
    left, right = (torch.randint(-2, 3, s, generator=g).double() for s in ((shape[0], rank), (rank, shape[1])))
    return (left @ right).to("cuda", dtype), left.cuda(), right.cuda()


def _low_rank_reference(left, right, steps, coefficients):
    """The iteration in the factors' small core, where no direction is empty: (X, Q, X_0)."""
    a, b, c = coefficients
    u, x = torch.linalg.qr(left)
    v, y = torch.linalg.qr(right.T)
    x = x @ y.T
    x = x0 = x / x.norm()
    eye = torch.eye(len(x), dtype=x.dtype, device=x.device)
    q = eye
    for _ in range(steps):
        g = x @ x.T
        p = a * eye + b * g + c * (g @ g)
        x, q = p @ x, p @ q
    whole = torch.eye(len(u), dtype=x.dtype, device=x.device)
    return u @ x @ v.T, a ** steps * (whole - u @ u.T) + u @ q @ u.T, u @ x0 @ v.T


@pytest.mark.parametrize("steps,coefficients", [(5, (A, B, C)), (10, (A, B, C)), (20, (A, B, C)), (100, (A, B, C)),
                                                (20, (1.5, -0.5, 0.0)), (100, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("shape,rank", [((7, 60), 1), ((16, 300), 2), ((500, 64), 8), ((200, 700), 8), ((700, 130), 3),
                                        ((300, 520), 4)])
def test_matrices_of_low_rank(shape, rank, steps, coefficients):
    """Directions that M does not have stay small for as many steps as are accepted. Q grows by a
    a step there, and each of its entries and each of the product's r sums is rounded in float32:
    the elementwise bound of this file's head, until a^steps reaches 2^20. From there on Q's norm is
    at most q = 2 / sqrt(2^-50 r) (a direction's value, at most 1.3, over the floor's root), and the
    error in norm e q (1 + sqrt(rank) + sqrt(r)): Q is q off the identity of the empty directions by
    its rounding e, by e sqrt(rank) off its part in the others, and r terms are added."""
    from causal_tuner.optim import orthogonalize
    m, left, right = _low_rank(shape, rank, torch.float32)
    got = orthogonalize(m, steps=steps, coefficients=coefficients)
    assert torch.isfinite(got).all()
    if shape[0] > shape[1]:
        got, left, right = got.T, right.T, left.T
    want, q, x0 = _low_rank_reference(left, right, steps, coefficients)
    r = min(shape)
    if coefficients[0] ** steps <= 2.0 ** 20:
        bound = 2 * (r + 4) * E32 * (q.abs() @ x0.abs())
        assert ((got.double() - want).abs() <= bound + E32 * want.abs()).all()
    else:
        most = 2 / (2.0 ** -50 * (-(-r // 32) * 32)) ** 0.5
        assert (got.double() - want).norm() <= E32 * most * (1 + rank ** 0.5 + r ** 0.5)


def test_muon_steps_of_low_rank_stay_finite():
    from causal_tuner.optim import FusedMuon
    shapes = [(64, 500), (200, 700), (16, 30)]
    params = [torch.nn.Parameter(_matrix(s, torch.bfloat16, seed=i) * 20) for i, s in enumerate(shapes)]
    before = [p.detach().clone() for p in params]
    for p, s in zip(params, shapes):
        p.grad = _low_rank(s, 2, torch.bfloat16)[0]
    FusedMuon(params, lr=0.02, weight_decay=0.0, ns_steps=100).step()
    for p, old in zip(params, before):
        assert torch.isfinite(p).all() and (p - old).norm() <= 0.02 * 3 * len(p) ** 0.5


def test_forward_mode_derivatives_are_refused():
    """Not dropped: host matrices carry them."""
    from torch.autograd import forward_ad
    from causal_tuner.optim import orthogonalize
    m = _matrix((20, 30), torch.float32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(m, torch.ones_like(m))
        for given in (dual, [m, dual]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                orthogonalize(given)
        host = orthogonalize(forward_ad.make_dual(m.cpu(), torch.ones(20, 30)))
        assert forward_ad.unpack_dual(host).tangent.any()
    _check(orthogonalize(m), m)


def test_sides_past_the_kernels_are_refused_by_name():
    from causal_tuner.optim import FusedMuon, orthogonalize
    for shape in ((16385, 16400), (1, (1 << 30) + 1)):
        with pytest.raises(NotImplementedError, match="up to 16384"):
            orthogonalize(torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(*shape))
    p = torch.nn.Parameter(torch.zeros(16385, 16385, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    optimizer = FusedMuon([p])
    with pytest.raises(NotImplementedError, match="up to 16384"):
        optimizer.step()
    assert not optimizer.state[p]


def _shifted(t, by):
    """The same tensor `by` elements into its storage: contiguous, at no 16-byte boundary."""
    return t.new_empty(t.numel() + by)[by:].view(t.shape).copy_(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
def test_muon_steps_of_every_kind_of_matrix(dtype, offset):
    """Two steps of one list: short sides of each of the Gram and last products' sizes up to 256 and
    past it, wide and tall, rows of four elements or not, and all of them at an odd element of
    their storage (parameter, gradient and momentum)."""
    from causal_tuner.optim import FusedMuon
    shapes = [(256, 300), (300, 256), (256, 1030), (200, 333), (333, 201), (129, 132), (300, 513), (513, 290), (290, 516),
              (33, 31), (1, 7), (7, 1), (60, 2051), (1030, 1100), (12, 20), (100, 64), (4, 4100)]
    params = [torch.nn.Parameter(_shifted(_matrix(s, dtype, seed=i) * 20, offset)) for i, s in enumerate(shapes)]
    lr, decay, mu = 0.02, 0.1, 0.9
    optimizer = FusedMuon(params, lr=lr, weight_decay=decay, momentum=mu)
    for i, (p, s) in enumerate(zip(params, shapes)):
        optimizer.state[p]["momentum_buffer"] = _shifted(_matrix(s, torch.float32, seed=50 + i), offset)
    u = torch.finfo(dtype).eps / 2
    for step in range(2):
        before = [p.detach().double() for p in params]
        held = [optimizer.state[p]["momentum_buffer"].double() for p in params]
        for i, p in enumerate(params):
            p.grad = _shifted(_matrix(shapes[i], dtype, seed=100 * step + i + 7), offset)
        kept = [p.grad.clone() for p in params]
        optimizer.step()
        for p, old, m, g in zip(params, before, held, kept):
            assert torch.equal(p.grad, g)
            buffer = optimizer.state[p]["momentum_buffer"]
            g = g.double()
            want = mu * m + (1 - mu) * g
            assert ((buffer.double() - want).abs() <= 4 * E32 * (mu * m.abs() + (1 - mu) * g.abs())).all(), tuple(p.shape)
            m = buffer.double()   # from here on with what the optimizer holds
            direction, bound = _reference(mu * m + (1 - mu) * g)
            rows, cols = p.shape
            factor = lr * max(1.0, rows / cols) ** 0.5
            want = old * (1 - lr * decay) - factor * direction
            allowed = factor * (bound + 3 * E32 * A ** 5 + 4 * E32 * direction.abs()) + 4 * E32 * old.abs()
            over = (p.double() - want).abs() - allowed - u * (want.abs() + allowed)
            assert over.max() <= 0, f"{tuple(p.shape)}: {over.max()} over a bound of {allowed.max()}"
