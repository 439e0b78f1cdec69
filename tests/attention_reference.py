"""Attention over packed records in float64 from its definition, with elementwise bounds on
what the kernels' roundings can change.

With u half a step of the tensors' type, e = 2^-24 and g = n e for a float32 sum of n terms
(first order, doubled below for what second-order terms and the exponential's last places add):

* a score is off by at most S = g_d |scale| sum |q||k| + 2 e |s| in its exponent, so p by
  S + max_j S relative (numerator and normalizer), plus u where it is rounded to bf16;
* o = sum p v / sum p, both of the rounded p, gains g_n + u (its own rounding); a rounding of
  p_j by r_j, |r_j| <= u, moves it by sum p_j r_j (v_j - o), at most u (sum p |v| + |o|);
* delta = do . o uses o and, for bf16, its rounding error, itself rounded to bf16 (off by u^2 |o|);
  its error is |do| . (the bound of that o) + g_d |do| . |o|;
* ds = p (do . v - delta) adds p times those errors and g_d |do| . |v|, and u |ds| where rounded;
* dq, dk, dv are sums of such terms, rounded once."""

import torch

E32 = 2.0 ** -24


def records_of(sizes, start=0, gap=0):
    out = []
    for n in sizes:
        out.append((start, start + n))
        start += n + gap
    return out


def reference(q, k, v, records, key_records, causal, scale, dout=None):
    """(values, bounds): lists of float64 tensors for out (and dq, dk, dv with `dout`)."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    pu = u if dtype == torch.bfloat16 else 0.0   # p and ds are rounded for bf16 inputs only
    q, k, v = (t.detach().double() for t in (q, k, v))
    dout = None if dout is None else dout.double()
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    shapes = [q, q, k, v]
    values, bounds = [torch.zeros_like(t) for t in shapes], [torch.zeros_like(t) for t in shapes]
    gd = (d + 4) * E32
    for (qa, qb), (ka, kb) in zip(records, key_records):
        lq, lk = qb - qa, kb - ka
        if not lq or not lk:
            continue
        gn, gr = (lk + 4) * E32, (lq * group + 4) * E32
        seen = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(lk - lq)
        empty = ~seen.any(-1, keepdim=True)
        for h in range(q.shape[1]):
            key, value = k[ka:kb, h // group], v[ka:kb, h // group]
            query = q[qa:qb, h]
            s = query @ key.T * scale
            off = 2 * (gd * scale * (query.abs() @ key.abs().T) + 2 * E32 * s.abs() + 4 * E32)
            s = s.masked_fill(~seen, float("-inf"))
            p = torch.where(empty, torch.zeros_like(s), torch.softmax(s, -1))
            off = torch.where(seen, off, torch.zeros_like(off))
            dp_rel = off + off.amax(-1, keepdim=True) + 2 * gn + pu
            o = p @ value
            bo = (p * dp_rel) @ value.abs() + 2 * gn * (p @ value.abs()) + pu * o.abs()
            taken = bo + (u * u if pu else u) * (o.abs() + bo)   # of what delta is made from
            bo = bo + u * (o.abs() + bo)
            values[0][qa:qb, h], bounds[0][qa:qb, h] = o, bo
            if dout is None:
                continue
            g = dout[qa:qb, h]
            delta = (g * o).sum(-1, keepdim=True)
            b_delta = (g.abs() * taken).sum(-1, keepdim=True) + gd * (g.abs() * o.abs()).sum(-1, keepdim=True)
            part = g @ value.T - delta
            ds = p * part
            b_ds = ds.abs() * (dp_rel + 4 * E32) + p * (1 + dp_rel) * (
                b_delta + 2 * gd * (g.abs() @ value.abs().T) + 2 * E32 * delta.abs()) * (1 + pu)
            values[1][qa:qb, h] += ds @ key * scale
            bounds[1][qa:qb, h] += scale * (b_ds @ key.abs() + 2 * gn * (ds.abs() @ key.abs()))
            values[2][ka:kb, h // group] += ds.T @ query * scale
            bounds[2][ka:kb, h // group] += scale * (b_ds.T @ query.abs() + 2 * gr * (ds.abs().T @ query.abs()))
            values[3][ka:kb, h // group] += p.T @ g
            bounds[3][ka:kb, h // group] += (p * dp_rel).T @ g.abs() + 2 * gr * (p.T @ g.abs())
    for i in (1, 2, 3):
        bounds[i] += u * (values[i].abs() + bounds[i]) + 2 * E32 * values[i].abs()
    n = 4 if dout is not None else 1
    return values[:n], bounds[:n]


def check(got, values, bounds, names=("out", "dq", "dk", "dv")):
    for name, x, y, b in zip(names, got, values, bounds):
        assert x.shape == y.shape, name
        off = (x.double() - y).abs()
        worst = (off - b).max().item() if off.numel() else 0.0
        assert torch.isfinite(x).all(), f"{name}: not finite"
        assert worst <= 1e-30, f"{name}: {worst} over its bound, at most {b.max().item()}; largest error {off.max()}"
