"""packed_attention (ct_attention_forward, ct_attention_backward) against float64 from the
definition, elementwise within bounds counted from its roundings (attention_reference.py)."""

import pytest
import torch

from attention_reference import check, records_of, reference

pytestmark = pytest.mark.gpu


def _tensors(tokens, key_tokens, heads, kv_heads, dim, dtype, seed=1, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, k, v = make(tokens, heads, dim), make(key_tokens, kv_heads, dim), make(key_tokens, kv_heads, dim)
    dout = make(tokens, heads, dim)
    return [t.requires_grad_(grad) for t in (q, k, v)] + [dout]


def _run(q, k, v, dout, layout, **kw):
    from causal_tuner.kernels.attention_cuda import packed_attention
    out = packed_attention(q, k, v, layout, **kw)
    if dout is None:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


def _case(sizes, key_sizes, heads, kv_heads, dim, dtype, causal, seed=1):
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    records, keys = records_of(sizes), records_of(key_sizes)
    q, k, v, dout = _tensors(sum(sizes), sum(key_sizes), heads, kv_heads, dim, dtype, seed)
    layout = AttentionLayout(records, "cuda", key_records=keys)
    got = _run(q, k, v, dout, layout, causal=causal)
    check(got, *reference(q, k, v, records, keys, causal, dim ** -0.5, dout))
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 1, 128), (6, 2, 64), (3, 3, 40), (5, 1, 96),
                                                (16, 1, 128), (2, 1, 8)])
def test_packed_records(heads, kv_heads, dim, causal, dtype):
    _case([1, 31, 0, 64, 65, 130], [1, 31, 0, 64, 65, 130], heads, kv_heads, dim, dtype, causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes,key_sizes", [
    ([1], [1]), ([1], [700]), ([1, 1, 1], [5, 129, 2048]), ([3, 1], [3, 64]), ([100], [1000]), ([33, 70], [97, 70]),
])
def test_queries_behind_a_cache(sizes, key_sizes, dtype):
    _case(sizes, key_sizes, 8, 2, 128, dtype, True)
    _case(sizes, key_sizes, 8, 2, 128, dtype, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_that_see_no_key(dtype):
    """More queries than keys: the first ones come before every key; records without keys or
    without queries."""
    out, dq, dk, dv = _case([70, 9, 0, 140], [10, 0, 12, 3], 4, 2, 64, dtype, True)
    assert not out[:60].any() and not dq[:60].any()
    assert not out[70:79].any() and not dk[10:22].any() and not dv[10:22].any()


def test_gradients_of_short_records_in_norm():
    """Where a row sees few keys, do . v - delta nearly cancels. ds, the results and the p behind
    delta are each rounded to bf16: uniform errors of at most half a step, 2^-8 / sqrt(3) in root
    mean square, together 2^-8 in norm; delta from the rounded output alone gives 0.0047."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    sizes = [1 + i % 4 for i in range(300)]
    records = records_of(sizes)
    q, k, v, dout = _tensors(sum(sizes), sum(sizes), 8, 8, 128, torch.bfloat16)
    got = _run(q, k, v, dout, AttentionLayout(records, "cuda"))
    want, _ = reference(q, k, v, records, records, True, 128 ** -0.5, dout)
    for x, y in zip(got, want):
        assert (x.double() - y).norm() <= 2.0 ** -8 * y.norm()
    lone = [a for a, b in records if b - a == 1]   # one key: p = 1, ds = 0
    assert got[1][lone].abs().max() < 1e-4


@pytest.mark.parametrize("dtype,length,heads,kv_heads,dim", [
    (torch.bfloat16, 1500, 4, 1, 128), (torch.bfloat16, 1111, 4, 4, 64), (torch.float32, 700, 3, 1, 128)])
def test_long_records(dtype, length, heads, kv_heads, dim):
    """Long enough that every pass runs many tiles and the key gradients are joined from parts."""
    _case([length, 300], [length, 300], heads, kv_heads, dim, dtype, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_offsets_and_batch_dimension(dtype):
    """Operands cut out of wider tensors (q, k and v side by side, heads first, odd element
    offsets that need a copy), a strided upstream gradient, and the [1, S, H, D] form."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    sizes, heads, dim = [37, 90], 4, 64
    records, tokens = records_of(sizes), sum(sizes)
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(tokens, (heads + 2) * dim, device="cuda", generator=g).to(dtype)
    side = [wide[:, :heads * dim].unflatten(1, (heads, dim)), wide[:, heads * dim:-dim].unflatten(1, (1, dim)),
            wide[:, -dim:].unflatten(1, (1, dim))]
    first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in side]      # heads outermost
    odd = []
    for t in side:
        buffer = torch.empty(t.numel() + 1, device="cuda", dtype=dtype)
        odd.append(buffer[1:].view(t.shape).copy_(t))                            # not 16-byte aligned
    dout = torch.randn(heads, tokens, dim, device="cuda", generator=g).to(dtype).transpose(0, 1)
    layout = AttentionLayout(records, "cuda")
    want = reference(*side, records, records, True, dim ** -0.5, dout)
    base = None
    for operands in (side, first, odd):
        leaves = [t.detach().requires_grad_(True) for t in operands]
        got = _run(*leaves, dout, layout)
        check(got, *want)
        base = base or got
        assert all(torch.equal(x, y) for x, y in zip(got, base))
    four = [t[None].requires_grad_(True) for t in side]
    out = packed_attention(*four, layout)
    assert out.shape == (1, tokens, heads, dim) and torch.equal(out[0], base[0])
    grads = torch.autograd.grad(out, four, dout[None])
    assert all(torch.equal(x[0], y) for x, y in zip(grads, base[1:]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_no_record_are_neither_read_nor_used(dtype):
    """NaN in front of, between and behind the records: outputs and gradients there are zero,
    everything else as without them."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    records, keys = [(3, 40), (45, 110)], [(5, 75), (80, 130)]
    q, k, v, dout = _tensors(120, 150, 4, 2, 128, dtype)
    inside = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in (120, 150)]
    for spans, rows in zip((records, keys), inside):
        for a, b in spans:
            rows[a:b] = True
    with torch.no_grad():
        for t, rows in ((q, inside[0]), (dout, inside[0]), (k, inside[1]), (v, inside[1])):
            t[~rows] = float("nan")
    got = _run(q, k, v, dout, AttentionLayout(records, "cuda", key_records=keys))
    check(got, *reference(q, k, v, records, keys, True, 128 ** -0.5, dout))
    for x, rows in zip(got, (inside[0], inside[0], inside[1], inside[1])):
        assert not x[~rows].any()


def test_scores_that_are_masked_or_minus_infinity():
    """Infinite scores of another record, and infinite values of a tile of keys that a row does
    not see, do not reach it."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    sizes = [200, 64]
    records = records_of(sizes)
    q, k, v, dout = _tensors(264, 264, 2, 1, 64, torch.bfloat16)
    with torch.no_grad():
        k[200:] = 3e38          # the second record overflows to infinite scores
        v[192:200] = float("inf")   # the first record's last tile of keys
    out = _run(q, k, v, None, AttentionLayout(records, "cuda"))[0]
    want, bound = reference(q[:192], k[:192], v[:192], [(0, 192)], [(0, 192)], True, 64 ** -0.5)
    check((out[:192],), want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_repeated_passes_are_bit_identical(dtype):
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    q, k, v, dout = _tensors(900, 900, 6, 2, 64, dtype)
    layout = AttentionLayout(records_of([500, 400]), "cuda")
    first = _run(q, k, v, dout, layout)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, _run(q, k, v, dout, layout)))


def test_far_offsets():
    """A cache past 4 GiB: keys and values of a record at its end."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    tokens, dim = (1 << 32) // 256 + 1000, 128
    cache = torch.zeros(2, tokens, 1, dim, device="cuda", dtype=torch.bfloat16)
    keys = [(10, 200), (tokens - 300, tokens)]
    q, k, v, _ = _tensors(5, 500, 4, 1, dim, torch.bfloat16, grad=False)
    cache[0, tokens - 300:], cache[1, tokens - 300:] = k[:300], v[:300]
    cache[0, 10:200], cache[1, 10:200] = k[300:490], v[300:490]
    layout = AttentionLayout([(0, 2), (2, 5)], "cuda", key_records=keys)
    out = _run(q, cache[0], cache[1], None, layout)
    near = torch.cat((k[300:490], k[:300])), torch.cat((v[300:490], v[:300]))
    check(out, *reference(q, *near, [(0, 2), (2, 5)], [(0, 190), (190, 490)], True, dim ** -0.5))


def test_keys_that_two_records_share():
    """A common prefix in the cache: allowed forward, refused backward."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    q, k, v, dout = _tensors(4, 300, 4, 2, 64, torch.bfloat16)
    records, keys = [(0, 1), (1, 4)], [(0, 200), (0, 300)]
    layout = AttentionLayout(records, "cuda", key_records=keys)
    out = packed_attention(q, k, v, layout)
    check((out.detach(),), *reference(q, k, v, records, keys, True, 64 ** -0.5))
    with pytest.raises(RuntimeError, match="overlap"):
        torch.autograd.grad(out, (q, k, v), dout)


def test_empty_inputs():
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    q, k, v, dout = _tensors(0, 7, 4, 2, 64, torch.bfloat16)
    out, dq, dk, dv = _run(q, k, v, dout, AttentionLayout([(0, 0)], "cuda", key_records=[(0, 7)]))
    assert out.shape == (0, 4, 64) and not dk.any() and not dv.any()
    q, k, v, dout = _tensors(5, 0, 4, 2, 64, torch.bfloat16)
    out, dq, dk, dv = _run(q, k, v, dout, AttentionLayout([(0, 5)], "cuda", key_records=[(0, 0)]))
    assert not out.any() and not dq.any() and dk.shape == (0, 2, 64)
    q, k, v, dout = _tensors(5, 5, 4, 2, 64, torch.bfloat16)
    got = _run(q, k, v, dout, AttentionLayout([], "cuda"))
    assert not any(x.any() for x in got)


def test_large_scores_stay_exact():
    """Rows whose maximum moves late and far: the running reference has to follow."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, dout = _tensors(400, 400, 2, 1, 64, torch.float32)
    with torch.no_grad():
        k.mul_(torch.linspace(0.1, 12, 400, device="cuda")[torch.randperm(400, device="cuda", generator=g)][:, None, None])
    records = [(0, 400)]
    layout = AttentionLayout(records, "cuda")
    for causal in (True, False):
        check(_run(q, k, v, dout, layout, causal=causal), *reference(q, k, v, records, records, causal, 0.125, dout))


def test_gradients_against_differences():
    """Central differences of the float32 forward along random directions. The loss is a sum of
    n values of about 1 and each forward value is good to about 2^-22: with a step h the quotient
    is off by 2^-22 sqrt(n) / h and by h^2 times third derivatives of order 1."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    q, k, v, dout = _tensors(50, 60, 4, 2, 32, torch.float32)
    layout = AttentionLayout([(0, 20), (20, 50)], "cuda", key_records=[(0, 25), (25, 60)])
    grads = _run(q, k, v, dout, layout)[1:]
    loss = lambda *t: (packed_attention(*t, layout).double() * dout.double()).sum().item()  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(9)
    h, base = 2.0 ** -7, [t.detach() for t in (q, k, v)]
    for i, grad in enumerate(grads):
        d = torch.randn(base[i].shape, device="cuda", generator=g)
        d = d / d.norm()
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(base)] for s in (1, -1))
        quotient = (loss(*up) - loss(*down)) / (2 * h)
        exact = (grad.double() * d.double()).sum().item()
        n = dout.numel()
        assert abs(quotient - exact) <= 2.0 ** -22 * n ** 0.5 / h * 4 + h * h * 4, (i, quotient, exact)


def test_two_streams_share_a_layout_that_dies_early():
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    records = records_of([300, 200])
    q, k, v, dout = _tensors(500, 500, 4, 1, 128, torch.bfloat16)
    want = reference(q, k, v, records, records, True, 128 ** -0.5, dout)
    torch.cuda.synchronize()
    layout = AttentionLayout(records, "cuda")
    results = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            results.append(_run(q, k, v, dout, layout))
    del layout
    noise = [torch.full((4096,), 7, device="cuda", dtype=torch.int32) for _ in range(20)]
    torch.cuda.synchronize()
    for got in results:
        check(got, *want)
    assert len(noise) == 20


def test_captured_passes_replay():
    """Forward and backward in one graph, replayed with new inputs between eager work; two graphs
    of one layout; the first call of a head layout is refused inside a capture."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    records = records_of([130, 70])
    layout = AttentionLayout(records, "cuda")
    held = [_tensors(200, 200, 4, 1, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    for q, k, v, dout in held:
        _run(q, k, v, dout, layout)
    torch.cuda.synchronize()
    graphs = []
    for q, k, v, dout in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _run(q, k, v, dout, layout)
        graphs.append((graph, got))
    for seed in range(3):
        for (q, k, v, dout), (graph, got) in zip(held, graphs):
            fresh = _tensors(200, 200, 4, 1, 128, torch.bfloat16, seed=10 + seed)
            with torch.no_grad():
                for t, x in zip((q, k, v, dout), fresh):
                    t.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            eager = _run(*fresh, layout)
            assert all(torch.equal(x, y) for x, y in zip(got, eager))
    unused = AttentionLayout(records, "cuda")
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            packed_attention(*held[0][:3], unused)
    torch.cuda.synchronize()
    check(_run(*held[0], layout), *reference(*held[0][:3], records, records, True, 128 ** -0.5, held[0][3]))


def test_device_refusals():
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    layout = AttentionLayout([(0, 4)], "cuda")
    make = lambda h, d, t=torch.bfloat16: torch.zeros(4, h, d, device="cuda", dtype=t)  # noqa: E731
    with pytest.raises(NotImplementedError):
        packed_attention(make(2, 64, torch.float16), make(1, 64, torch.float16), make(1, 64, torch.float16), layout)
    for dim in (136, 12, 256):
        with pytest.raises(ValueError, match="head_dim"):
            packed_attention(make(2, dim), make(1, dim), make(1, dim), layout)
    with pytest.raises(ValueError, match="layout is on"):
        packed_attention(make(2, 64), make(1, 64), make(1, 64), AttentionLayout([(0, 4)], "cpu"))
    with pytest.raises(ValueError, match="different devices"):
        packed_attention(make(2, 64), make(1, 64).cpu(), make(1, 64), layout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes,key_sizes", [([200], [200]), ([1, 3], [700, 900])])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("exponent", [14, 16, 24, 34, 100])
def test_scores_of_any_size(exponent, dim, sizes, key_sizes, dtype):
    """Scores s = +-2^exponent k / 8 of whole k, so that each row's softmax is 1 at its largest
    score or 1/2 at two equal ones and 0 elsewhere: a float32 sum of m and log2 of the
    denominator would lose the latter from scores of 2^16 on. v and dout are -1, 0 or 1, so all
    sums and ds = (dp_1 - dp_2) / 4 (at most 8 bits) are exact; what is left is the results' rounding and the last
    places of the exponential and the logarithm."""
    from causal_tuner.kernels.attention_cuda import AttentionLayout
    tokens, key_tokens, heads = sum(sizes), sum(key_sizes), 4
    records, keys = records_of(sizes), records_of(key_sizes)
    g = torch.Generator().manual_seed(exponent)
    if len(sizes) == 1:
        number = torch.arange(key_tokens) // 2 + 1
    else:
        number = torch.randint(1, 100, (key_tokens,), generator=g)
        for start, _ in keys:
            number[[start + 5, start + 420]], number[[start + 7, start + 555]] = 200, 0
    q = torch.zeros(tokens, heads, dim)
    q[:, :, 0] = 2.0 ** exponent * torch.tensor([1.0, -1.0, 1.0, -1.0])
    k = torch.zeros(key_tokens, 1, dim)
    k[:, 0, 0] = number
    v, dout = (torch.randint(-1, 2, s, generator=g).float() for s in ((key_tokens, 1, dim), (tokens, heads, dim)))
    leaves = [t.to("cuda", dtype).requires_grad_(True) for t in (q, k, v)]
    got = _run(*leaves, dout.to("cuda", dtype), AttentionLayout(records, "cuda", key_records=keys), scale=0.125)
    want, _ = reference(*leaves, records, keys, True, 0.125, dout.cuda())
    assert not want[1].any() and want[2].any()
    u = torch.finfo(dtype).eps / 2
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        assert ((x.double() - y).abs() <= (u + 8 * 2.0 ** -24) * y.abs()).all(), name


def test_forward_mode_derivatives_are_refused():
    """Not dropped: with and without a gradient asked for, and of the upstream gradient."""
    from torch.autograd import forward_ad
    from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention
    q, k, v, dout = _tensors(20, 20, 2, 1, 64, torch.float32, grad=False)
    layout = AttentionLayout([(0, 20)], "cuda")
    want = packed_attention(q, k, v, layout)
    with forward_ad.dual_level():
        for i in range(3):
            operands = [q, k, v]
            operands[i] = forward_ad.make_dual(operands[i], torch.ones_like(operands[i]))
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    packed_attention(*operands, layout)
        assert torch.equal(packed_attention(q, k, v, layout), want)
        leaf = q.clone().requires_grad_(True)
        out = packed_attention(leaf, k, v, layout)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(dout, dout))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: packed_attention(t, k, v, layout), (q,), (q,))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,sizes,key_sizes", [
    (24, 1, 64, [1, 70, 129], [1, 70, 129]), (32, 1, 128, [65, 40], [65, 40]), (33, 1, 64, [9, 50], [30, 50]),
    (48, 1, 128, [33, 3, 60], [33, 3, 60]), (72, 2, 40, [21, 30], [21, 45]), (130, 1, 64, [5, 17], [5, 80]),
    (64, 64, 16, [40], [40])])
def test_many_heads_to_a_key_value_head(heads, kv_heads, dim, sizes, key_sizes, dtype):
    """Groups as large as a step of 32 rows, which they divide, and past it; past a tile of 128."""
    _case(sizes, key_sizes, heads, kv_heads, dim, dtype, True)
