"""orthogonalize and FusedMuon without a device: host tensors, refusals, ct_muon_plan's shares."""

import ctypes
import random

import pytest
import torch

from causal_tuner.kernels import _native
from causal_tuner.optim import FusedMuon, orthogonalize


def _iterate(m, steps=5):
    a, b, c = 3.4445, -4.7750, 2.0315
    x = m.double() / max(float(m.double().norm()), 1e-7)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + b * g @ x + c * g @ (g @ x)
    return x


@pytest.mark.parametrize("shape", [(3, 7), (7, 3), (5, 5), (1, 4), (4, 1)])
def test_host_matrices(shape):
    m = torch.randn(*shape)
    want = _iterate(m) if shape[0] <= shape[1] else _iterate(m.T).T
    torch.testing.assert_close(orthogonalize(m).double(), want, rtol=1e-6, atol=1e-7)
    one, two = orthogonalize([m, m.bfloat16()])
    assert one.dtype == torch.float32 and two.dtype == torch.bfloat16
    assert orthogonalize(torch.empty(0, 3)).shape == (0, 3)


def test_refusals():
    with pytest.raises(ValueError, match="not a matrix"):
        orthogonalize(torch.zeros(3))
    with pytest.raises(ValueError, match="floating"):
        orthogonalize(torch.zeros(3, 3, dtype=torch.int32))
    for options in ({"steps": 0}, {"steps": 101}, {"steps": 2.5}, {"eps": -1.0}, {"eps": float("nan")},
                    {"coefficients": (1.0, float("inf"), 0.0)}):
        with pytest.raises(ValueError):
            orthogonalize(torch.zeros(3, 3), **options)
    p = torch.nn.Parameter(torch.zeros(3, 3))
    for options in ({"lr": -1.0}, {"momentum": -0.1}, {"momentum": 1.5}, {"weight_decay": -1.0}, {"ns_steps": 0},
                    {"adjust_lr_fn": "else"}):
        with pytest.raises(ValueError):
            FusedMuon([p], **options)
    with pytest.raises(ValueError, match="matrices only"):
        FusedMuon([torch.nn.Parameter(torch.zeros(3))])
    p.grad = torch.zeros(3, 3)
    with pytest.raises(NotImplementedError):
        FusedMuon([p]).step()


def _plan(shapes):
    lib, kinds = _native.library(), _native.CT_MUON_KINDS
    table = (_native.MuonMatrix * len(shapes))()
    for row, (rows, cols) in zip(table, shapes):
        row.rows, row.cols = rows, cols
    counts, nbytes = (ctypes.c_int64 * kinds)(), ctypes.c_int64()
    assert lib.ct_muon_plan(table, len(shapes), None, 0, counts, ctypes.byref(nbytes)) == 0
    entries = torch.zeros(max(sum(counts), 1), 8, dtype=torch.int32)
    if sum(counts):
        assert lib.ct_muon_plan(table, len(shapes), entries.data_ptr(), sum(counts) - 1, counts, ctypes.byref(nbytes)) == -5
    assert lib.ct_muon_plan(table, len(shapes), entries.data_ptr(), sum(counts), counts, ctypes.byref(nbytes)) == 0
    rows, kinds_of = entries.tolist(), []
    for count in counts:
        kinds_of.append(rows[:count])
        rows = rows[count:]
    return table, kinds_of, nbytes.value


def test_plans_cover_every_matrix_once():
    """Ranges of the long side follow one another in the Gram and the last products; partials and
    buffers lie one behind the other in the workspace, behind the table."""
    rng = random.Random(1)
    for _ in range(60):
        shapes = [(rng.choice([1, 5, 16, 40, 100, 255, 256, 257, 600]), rng.choice([1, 7, 64, 300, 3000, 9000]))
                  for _ in range(rng.randint(1, 30))]
        table, (gram, tiles, momentum, join, stage, small, last), nbytes = _plan(shapes)
        spans = [(0, len(shapes) * ctypes.sizeof(_native.MuonMatrix) / 8)]
        for i, shape in enumerate(shapes):
            r, width = min(shape), max(shape)
            rp, t = -(-r // 32) * 32, -(-r // 16)
            for items, used in ((gram, r <= 256), (tiles, r > 256), (last, True)):
                pairs = {}
                for m, a, b, lo, hi, slot, *_ in items:
                    if m == i:
                        pairs.setdefault((a, b), []).append((lo, hi, slot))
                assert bool(pairs) == used
                for ranges in pairs.values():
                    ranges.sort()
                    assert ranges[0][0] == 0 and ranges[-1][1] == width
                    assert all(x[1] == y[0] for x, y in zip(ranges, ranges[1:]))
                    if items is not last:
                        assert [x[2] for x in ranges] == list(range(table[i].splits))
            blocks = sorted((a, b) for m, a, b, *_ in stage if m == i)
            assert blocks == ([] if r <= 64 else [(a, b) for a in range(rp // 32) for b in range(a + 1)])
            assert sum(m == i for m, *_ in small) == (r <= 64)
            assert sum(m == i for m, *_ in join) == (0 if r <= 64 else (rp // 16) * (rp // 16 + 1) // 2)
            head = 2 if r <= 256 else (-(-r // 64) + 1) // 2 * 2
            spans.append((table[i].parts, table[i].parts + table[i].splits * (head + t * (t + 1) // 2 * 256)))
            spans.append((table[i].scratch, table[i].scratch + 2 + (0 if r <= 64 else 5 * rp * rp) + rp * rp // 2))
        spans.sort()
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and spans[-1][1] * 8 <= nbytes


def test_abi_refusals():
    lib = _native.library()
    table = (_native.MuonMatrix * 1)()
    counts, nbytes = (ctypes.c_int64 * _native.CT_MUON_KINDS)(), ctypes.c_int64()
    for rows, cols in ((0, 4), (4, 0), (-1, 3), (20000, 20000), (4, 1 << 31)):
        table[0].rows, table[0].cols = rows, cols
        assert lib.ct_muon_plan(table, 1, None, 0, counts, ctypes.byref(nbytes)) == -2
    assert lib.ct_muon_plan(None, 1, None, 0, counts, ctypes.byref(nbytes)) == -1
    assert lib.ct_muon_plan(table, -1, None, 0, counts, ctypes.byref(nbytes)) == -2
    table[0].rows, table[0].cols = 4, 6
    assert lib.ct_muon_plan(table, 1, None, 0, counts, ctypes.byref(nbytes)) == 0
    options = _native.MuonOptions(steps=5)
    call = lambda plan=256, dt=0, o=options, ws=256, n=1 << 30: lib.ct_muon(  # noqa: E731
        table, 1, plan, counts, dt, ctypes.byref(o), ws, n, nbytes.value, None)
    assert call() == -1                       # no param
    table[0].param = table[0].grad = 256
    assert call(dt=1) == -3 and call(plan=None) == -1 and call(plan=264) == -1
    assert call(ws=None) == -5 and call(n=8) == -5
    assert call(o=_native.MuonOptions(steps=0)) == -2 and call(o=_native.MuonOptions(steps=101)) == -2
    assert call(o=_native.MuonOptions(steps=5, update=1)) == -1   # no momentum


def test_groups_of_their_own_are_checked_and_refused_ones_left_out():
    make = lambda *s: torch.nn.Parameter(torch.zeros(*s))  # noqa: E731
    first = make(3, 4)
    optimizer = FusedMuon([first], lr=0.1)
    for group in ({"params": [make(3, 4), make(3)]}, {"params": [make(3, 4)], "lr": -1.0},
                  {"params": [make(3, 4)], "momentum": 2.0}, {"params": [make(3, 4)], "weight_decay": -1.0},
                  {"params": [make(3, 4)], "adjust_lr_fn": "else"}, {"params": [make(3, 4)], "ns_steps": 0},
                  {"params": [make(3, 4)], "eps": -1.0}):
        with pytest.raises(ValueError):
            optimizer.add_param_group(group)
        assert len(optimizer.param_groups) == 1 and optimizer.param_groups[0]["params"] == [first]
        with pytest.raises(ValueError):
            FusedMuon([group])
    second = make(4, 3)
    optimizer.add_param_group({"params": (p for p in [second]), "adjust_lr_fn": "match_rms_adamw"})
    assert optimizer.param_groups[1]["params"] == [second] and optimizer.param_groups[1]["lr"] == 0.1


def test_the_largest_sides():
    """The sizes that the Python calls refuse by name are those that ct_muon_plan refuses."""
    from causal_tuner.optim import _refuse_large
    lib = _native.library()
    counts, nbytes = (ctypes.c_int64 * _native.CT_MUON_KINDS)(), ctypes.c_int64()
    table = (_native.MuonMatrix * 1)()
    for shape, fits in (((16384, 16384), True), ((16385, 16385), False), ((1, 1 << 30), True), ((1 << 30, 1), True),
                        ((1, (1 << 30) + 1), False), (((1 << 30) + 1, 1), False), ((16384, 20000), True)):
        table[0].rows, table[0].cols = shape
        assert lib.ct_muon_plan(table, 1, None, 0, counts, ctypes.byref(nbytes)) == (0 if fits else -2), shape
        if fits:
            _refuse_large("orthogonalize", shape)
        else:
            with pytest.raises(NotImplementedError, match="up to 16384"):
                _refuse_large("orthogonalize", shape)
