"""packed_attention without a device: the host path against float64 from the definition, its
gradients, the layout's checks and the C ABI's refusals and plans."""

import ctypes
import random

import pytest
import torch

from attention_reference import check, records_of, reference
from causal_tuner.kernels import _native
from causal_tuner.kernels.attention_cuda import AttentionLayout, packed_attention


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("sizes,key_sizes", [([1, 31, 0, 64], [1, 31, 0, 64]), ([70, 9, 0, 14], [10, 0, 12, 30])])
def test_host_path(sizes, key_sizes, causal, dtype):
    make = lambda n, h: torch.randn(n, h, 24).to(dtype).requires_grad_(True)  # noqa: E731
    q, k, v = make(sum(sizes), 6), make(sum(key_sizes), 2), make(sum(key_sizes), 2)
    dout = torch.randn(sum(sizes), 6, 24).to(dtype)
    records, keys = records_of(sizes), records_of(key_sizes)
    out = packed_attention(q, k, v, AttentionLayout(records, "cpu", key_records=keys), causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    check((out.detach(), *grads), *reference(q, k, v, records, keys, causal, 24 ** -0.5, dout))


def test_list_of_records_and_batch_dimension():
    q, k, v = torch.randn(1, 9, 4, 8), torch.randn(1, 9, 1, 8), torch.randn(1, 9, 1, 8)
    out = packed_attention(q, k, v, [(0, 4), (4, 9)], scale=0.3)
    check((out[0],), *reference(q[0], k[0], v[0], [(0, 4), (4, 9)], [(0, 4), (4, 9)], True, 0.3))


def test_host_path_in_double():
    """Double tensors are worked on in double: against differences, with a shared head and queries
    that see no key."""
    q, k, v = (torch.randn(n, h, 3, dtype=torch.float64, requires_grad=True) for n, h in ((7, 4), (6, 2), (6, 2)))
    layout = AttentionLayout([(0, 4), (4, 7)], "cpu", key_records=[(0, 2), (2, 6)])
    assert torch.autograd.gradcheck(lambda *t: packed_attention(*t, layout), (q, k, v))


def test_refusals():
    with pytest.raises(ValueError, match="overlap"):
        AttentionLayout([(0, 5), (4, 8)], "cpu")
    with pytest.raises(ValueError, match="span"):
        AttentionLayout([(5, 3)], "cpu")
    with pytest.raises(ValueError, match="span"):
        AttentionLayout([(-1, 3)], "cpu")
    with pytest.raises(ValueError, match="keys for"):
        AttentionLayout([(0, 5)], "cpu", key_records=[(0, 2), (2, 5)])
    q, k = torch.zeros(5, 4, 8), torch.zeros(5, 2, 8)
    bad = [(q, torch.zeros(5, 3, 8), torch.zeros(5, 3, 8), {}), (q, torch.zeros(5, 2, 16), torch.zeros(5, 2, 16), {}),
           (q, k, torch.zeros(6, 2, 8), {}), (q[0], k, k, {}), (q, k.double(), k.double(), {}),
           (q, torch.zeros(5, 0, 8), torch.zeros(5, 0, 8), {}), (q, k, k, {"scale": 0.0}), (q, k, k, {"scale": -1.0}),
           (q, k, k, {"scale": float("nan")}), (q, k, k, {"scale": float("inf")}), (q, k, k, {"scale": 1e-60}),
           (q, k, k, {"scale": 3e38}), (q.int(), k.int(), k.int(), {}),
           (torch.zeros(5, 4, 0), torch.zeros(5, 2, 0), torch.zeros(5, 2, 0), {})]
    for a, b, c, options in bad:
        with pytest.raises(ValueError):
            packed_attention(a, b, c, [(0, 5)], **options)
    with pytest.raises(ValueError, match="reach to"):
        packed_attention(q, k, k, [(0, 6)])
    with pytest.raises(ValueError, match="reach to"):
        packed_attention(q, k, k, AttentionLayout([(0, 5)], "cpu", key_records=[(0, 9)]))


def _plan(kind, records, heads, kv_heads, dim, causal, dtype=_native.CT_BF16):
    table = torch.tensor(records, dtype=torch.int64).reshape(-1, 4)
    counts = (ctypes.c_int64 * 4)()
    fixed = (kind, table.data_ptr(), len(records), heads, kv_heads, dim, dtype, int(causal))
    lib = _native.library()
    assert lib.ct_attention_plan(*fixed, None, 0, counts) == 0
    size = counts[0] + counts[1] + counts[3]
    entries = torch.zeros(max(size, 1), 8, dtype=torch.int32)
    if size:
        assert lib.ct_attention_plan(*fixed, entries.data_ptr(), size - 1, counts) == -5
    assert lib.ct_attention_plan(*fixed, entries.data_ptr(), size, counts) == 0
    rows = entries.tolist()
    return rows[:counts[0]], rows[counts[0]:counts[0] + counts[1]], rows[counts[0] + counts[1]:size], counts[2]


@pytest.mark.parametrize("kind", [_native.CT_ATTENTION_FORWARD, _native.CT_ATTENTION_ROWS, _native.CT_ATTENTION_KEYS])
def test_plans_cover_every_tile_once(kind):
    """Every tile of 128 rows or keys: its pieces follow one another from its first to its last
    key or row, cut ones have partials in order and joins for all their rows; every piece belongs
    to one workgroup."""
    rng = random.Random(kind)
    for _ in range(150):
        kv_heads, group = rng.choice([1, 2, 8]), rng.choice([1, 3, 4, 16, 33])
        causal, records, q, k = rng.random() < 0.7, [], 0, 0
        for _ in range(rng.randint(0, 5)):
            lq = rng.choice([0, 1, 3, 77, 300, 2000])
            lk = rng.choice([lq, 0, 1, 33, lq + 500, 5000, 20000])
            records.append((q, lq, k, lk))
            q, k = q + lq, k + lk
        pieces, joins, groups, slots = _plan(kind, records, group * kv_heads, kv_heads, rng.choice([64, 128]), causal)
        assert sorted(i for first, count, *_ in groups for i in range(first, first + count)) == list(range(len(pieces)))
        assert sorted(p[4] for p in pieces if p[4] >= 0) == list(range(slots))
        tiles, joined = {}, {}
        for record, begin, lo, hi, slot, *_ in pieces:
            tiles.setdefault((record, begin), []).append((lo, hi, slot))
        for j in joins:
            joined.setdefault((j[0], j[1]), []).append(j)
        for r, (_, lq, _, lk) in enumerate(records):
            rows = lq * group
            span = lk if kind == _native.CT_ATTENTION_KEYS else rows
            for begin in range(0, span, 128):
                parts = sorted(tiles.pop((r, begin)))
                assert all(a[1] == b[0] and a[2] + 1 == b[2] for a, b in zip(parts, parts[1:]))
                if kind == _native.CT_ATTENTION_KEYS:
                    first = max(0, begin - (lk - lq)) * group if causal else 0
                    assert parts[0][0] <= first or parts[0][0] == rows
                    assert parts[-1][1] == rows
                else:
                    last = (min(rows, begin + 128) - 1) // group
                    assert parts[0][0] == 0
                    assert parts[-1][1] == (min(lk, max(0, last + 1 + lk - lq)) if causal else lk)
                own = sorted(joined.pop((r, begin), []), key=lambda j: j[4])
                if len(parts) == 1:
                    assert not own and parts[0][2] == -1
                    continue
                at = 0
                for j in own:
                    assert (j[2], j[3]) == (parts[0][2], len(parts)) and j[4] == at and j[5] > 0
                    at += j[5]
                assert at == min(128, span - begin)
        assert not tiles and not joined


def test_abi_refusals():
    lib = _native.library()
    counts = (ctypes.c_int64 * 4)()
    table = torch.tensor([[0, 5, 0, 5]], dtype=torch.int64)
    plan = lambda kind=0, t=table, n=1, h=4, kv=2, d=64, dt=2: lib.ct_attention_plan(  # noqa: E731
        kind, t.data_ptr() if t is not None else None, n, h, kv, d, dt, 1, None, 0, counts)
    assert plan() == 0
    assert plan(kind=3) == -2 and plan(h=3) == -2 and plan(kv=0) == -2 and plan(d=12) == -2 and plan(d=136) == -2
    assert plan(dt=1) == -3 and plan(t=None) == -1
    assert plan(t=torch.tensor([[0, -1, 0, 5]])) == -2 and plan(t=torch.tensor([[0, 5, 0, 1 << 40]])) == -2
    assert lib.ct_attention_plan(0, table.data_ptr(), 1, 4, 2, 64, 2, 1, None, 0, None) == -1
    good = dict(q=256, k=256, v=256, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, records=256,
                heads=4, kv_heads=2, head_dim=64, dtype=_native.CT_BF16, causal=1, scale=0.125)
    plan()
    # one workgroup is planned, so an output is needed; every field out of range is refused first
    forward = lambda out=None, **bad: lib.ct_attention_forward(  # noqa: E731
        ctypes.byref(_native.Attention(**{**good, **bad})), None, counts, out, None, None, 0, None)
    assert forward() == -1
    assert lib.ct_attention_forward(None, None, counts, None, None, None, 0, None) == -1
    assert forward(dtype=_native.CT_F16) == -3
    for bad in (dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(head_dim=20), dict(heads=5),
                dict(q_token=257), dict(k_head=-64), dict(k_token=1 << 24), dict(q_token=1 << 30)):
        assert forward(**bad) == -2, bad
    for bad in (dict(q=None), dict(k=264), dict(records=None)):
        assert forward(**bad) == -1, bad
    counts[2] = 3
    assert lib.ct_attention_forward(ctypes.byref(_native.Attention(**good)), 256, counts, 256, None, None, 0, None) == -5
    counts[0] = -1
    assert forward() == -2


def test_host_tangents():
    """Host tensors carry forward-mode derivatives: against differences."""
    from torch.autograd import forward_ad
    q, k, v = (torch.randn(6, h, 4, dtype=torch.float64) for h in (4, 2, 2))
    along, h = torch.randn_like(k), 1e-6
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(packed_attention(q, forward_ad.make_dual(k, along), v, [(0, 6)])).tangent
    up, down = (packed_attention(q, k + s * h * along, v, [(0, 6)]) for s in (1, -1))
    torch.testing.assert_close(tangent, (up - down) / (2 * h), rtol=1e-6, atol=1e-8)


def test_decoder_records():
    """The decoder's positions restart at each record as listed: records out of order or with keys
    of others are refused, not attended to with other rows' positions."""
    from causal_tuner.modeling import decoder
    config = decoder.DecoderConfig(hidden_size=16, num_attention_heads=2, head_dim=8, intermediate_size=16,
                                   num_hidden_layers=1, vocab_size=10, attention="packed")
    plain = decoder.DecoderConfig(**{**vars(config), "attention": "sdpa"})
    q, k, v = torch.randn(1, 9, 2, 8), torch.randn(1, 9, 1, 8), torch.randn(1, 9, 1, 8)
    want = packed_attention(q, k, v, [(0, 4), (4, 4), (4, 9)])
    for records in ([(0, 4), (4, 4), (4, 9)], [(0, 4), (4, 9), (0, 0)], AttentionLayout([(0, 4), (4, 9)], "cpu")):
        assert torch.equal(decoder._attention(q, k, v, records, config), want)
    for records in ([(4, 9), (0, 4)], [(0, 4), (4, 8)], [(0, 4), (5, 9)]):
        with pytest.raises(ValueError, match="cover the sequence"):
            decoder._attention(q, k, v, records, config)
    others = AttentionLayout([(0, 4), (4, 9)], "cpu", key_records=[(0, 4), (0, 9)])
    for c in (config, plain):
        with pytest.raises(ValueError, match="key_records"):
            decoder._attention(q, k, v, others, c)
        assert decoder.packed_records([(0, 9)], c, "cpu") is not None
