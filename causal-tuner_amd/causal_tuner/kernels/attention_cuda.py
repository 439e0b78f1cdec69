"""Attention over packed records on gfx950, forward and backward.

The reference runs its attention through a library (kernels/attention.py:16-93: a layout
prepared once per batch, then one varlen call per layer); here `AttentionLayout` is that
layout and `packed_attention` the call, on the HIP kernels ct_attention_forward and
ct_attention_backward.

    layout = AttentionLayout([(0, 1411), (1411, 2217)], "cuda")     # once per batch
    out = packed_attention(q, k, v, layout)                         # q [S, H, D], k, v [S, H_kv, D]

Each record's queries attend to its own keys: softmax(scale q k^T) v, causal by default. With
`key_records` the keys of a record lie elsewhere and may be more than its queries; the
queries are then the last of them (causal: query i of L_q sees keys 0 .. i + L_k - L_q), the
form of a prompt that continues a cache and, with one query per record, of writing answers
token by token. A query that sees no key gives zeros, and no gradient. The scores, their
statistics and every sum are float32; the probabilities and their gradients are rounded to
bf16 for bf16 inputs, whose backward keeps the output's rounding error, a tensor of the output's
size. Repeated calls, backward included, are bit-identical.

A masked score counts as minus infinity whatever it holds, and rows of no record are never
read. Inside a record, a key or value that is not finite makes NaN of every row whose tile of
64 keys holds it, masked or not (0 x inf), as the plain product of probabilities and values
does.

Host tensors take the same formulas in torch operations.
"""

import ctypes
import math

import torch

from . import _native

_PASSES = {"forward": _native.CT_ATTENTION_FORWARD, "rows": _native.CT_ATTENTION_ROWS,
           "keys": _native.CT_ATTENTION_KEYS}
_ENTRY = 8                 # int32 per plan entry
_MAX_PITCH = 1 << 24       # bytes between two tokens of k and v
_MAX_SPAN = (1 << 31) - 1024


def _spans(records, name):
    spans = []
    for record in records:
        start, stop = (int(x) for x in record)
        if not 0 <= start <= stop:
            raise ValueError(f"{name}: ({start}, {stop}) is not a span")
        spans.append((start, stop))
    return spans


def _disjoint(spans):
    ordered = sorted(s for s in spans if s[0] < s[1])
    return all(a[1] <= b[0] for a, b in zip(ordered, ordered[1:]))


class _Plan:
    """One pass's shares of work: their device address, the counts and the partials' bytes."""

    __slots__ = ("entries", "counts", "workspace")

    def __init__(self, entries, counts, workspace):
        self.entries, self.counts, self.workspace = entries, counts, workspace


class _Tables:
    """The device tables of one head layout: the records and every pass's plan, in one copy."""

    __slots__ = ("device_copy", "stream", "records", "forward", "rows", "keys")

    def use(self, stream):
        """Keeps the copy's memory from other use until this stream's work is done with it."""
        if stream != self.stream and not torch.cuda.is_current_stream_capturing():
            self.device_copy.record_stream(torch.cuda.current_stream(self.device_copy.device))


class AttentionLayout:
    """Packed records of a batch as the attention kernels take them, for one device.

    `records` are the queries' (start, stop) spans; `key_records` (default: the same) the
    spans of each record's keys. Queries may not belong to two records; keys may, but then
    there is no backward. Rows of no record are allowed: their outputs and gradients are zero.

    A layout is made once per batch and serves every layer. The device tables that a call
    needs (they depend on the head layout) are made at the first call with that head layout and
    kept: one small copy, which the host waits for, so the tables are valid on every stream.
    That first call cannot be made inside a graph capture, and a captured graph needs the
    layout kept as long as itself.
    """

    def __init__(self, records, device, *, key_records=None):
        self.records = _spans(records, "records")
        self.key_records = self.records if key_records is None else _spans(key_records, "key_records")
        if len(self.records) != len(self.key_records):
            raise ValueError(f"{len(self.records)} records, but keys for {len(self.key_records)}")
        if not _disjoint(self.records):
            raise ValueError("records overlap")
        self.keys_disjoint = self.key_records is self.records or _disjoint(self.key_records)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.tokens = max((stop for _, stop in self.records), default=0)
        self.key_tokens = max((stop for _, stop in self.key_records), default=0)
        # whether the records follow one another, each with its own rows as keys
        filled = [r for r in self.records if r[0] < r[1]]
        self.in_order = self.key_records == self.records and filled == sorted(filled)
        # whether every row of the spans' range belongs to a record
        self.whole = sum(b - a for a, b in self.records) == self.tokens
        self.keys_whole = self.keys_disjoint and sum(b - a for a, b in self.key_records) == self.key_tokens
        self._host = torch.tensor([[a, b - a, c, d - c] for (a, b), (c, d) in zip(self.records, self.key_records)],
                                  dtype=torch.int64).reshape(-1, 4)
        self._tables = {}

    def tables(self, heads, kv_heads, head_dim, dtype, causal):
        key = (heads, kv_heads, head_dim, dtype, causal)
        tables = self._tables.get(key)
        if tables is None:
            tables = self._tables[key] = self._make_tables(*key)
        return tables

    def _make_tables(self, heads, kv_heads, head_dim, dtype, causal):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AttentionLayout: the first call with a head layout makes its tables and cannot be "
                               "captured; run it once before the capture")
        lib = _native.library()
        parts, plans, at = [self._host.view(torch.int32).reshape(-1, _ENTRY)], {}, len(self._host)
        for name, code in _PASSES.items():
            counts = (ctypes.c_int64 * 4)()
            fixed = (code, _native.ptr(self._host), len(self._host), heads, kv_heads, head_dim, _native.dtype_code(dtype),
                     int(causal))
            _native.check(lib.ct_attention_plan(*fixed, None, 0, counts), "ct_attention_plan")
            size = counts[0] + counts[1] + counts[3]
            entries = torch.empty(size, _ENTRY, dtype=torch.int32)
            if size:
                _native.check(lib.ct_attention_plan(*fixed, _native.ptr(entries), size, counts), "ct_attention_plan")
            parts.append(entries)
            plans[name] = (at, counts, lib.ct_attention_workspace(code, counts[2], kv_heads, head_dim))
            at += size
        tables = _Tables()
        with torch.cuda.device(self.device):
            tables.device_copy = torch.cat(parts).to(self.device)
            tables.stream = _native.stream_of(tables.device_copy)
        tables.records = tables.device_copy.data_ptr()
        for name, (start, counts, workspace) in plans.items():
            setattr(tables, name, _Plan(tables.records + start * 4 * _ENTRY, counts, workspace))
        return tables


def _strided(t, tokens_at_once, heads):
    """`t` [tokens, heads, head_dim] in a form that the kernels take: itself, or a contiguous
    copy where an element stride, an alignment or a span of strides is not theirs."""
    size = t.element_size()
    token, head, unit = t.stride()
    if (unit != 1 or token * size % 16 or head * size % 16 or t.data_ptr() % 16 or token < 0 or head < 0
            or token * size > _MAX_PITCH or tokens_at_once * token * size + heads * head * size >= _MAX_SPAN):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _operands(q, k, v, tables, causal, scale, rest):
    q_token, q_head, _ = q.stride()
    k_token, k_head, _ = k.stride()
    v_token, v_head, _ = v.stride()
    return _native.Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), q_token, q_head, k_token, k_head, v_token, v_head,
                             tables.records, q.shape[1], k.shape[1], q.shape[2], _native.dtype_code(q.dtype), causal,
                             scale, _native.ptr(rest))


def _forward(q, k, v, layout, causal, scale, keep_stats):
    """(q, k, v as the kernels read them, out, its rounding error or None, stats or None)."""
    tokens, heads, head_dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    q, k, v = _strided(q, 64 // group + 2, group), _strided(k, 64, 0), _strided(v, 64, 0)
    work = layout.tokens and layout.key_tokens   # else there is nothing but zeros
    fresh = torch.empty if work and layout.whole and layout.tokens == tokens else torch.zeros
    out = fresh((tokens, heads, head_dim), dtype=q.dtype, device=q.device)
    rest = torch.empty_like(out) if keep_stats and q.dtype == torch.bfloat16 else None
    stats = torch.empty((tokens, heads, 2), dtype=torch.float32, device=q.device) if keep_stats else None
    if work:
        tables = layout.tables(heads, kv_heads, head_dim, q.dtype, causal)
        plan, stream = tables.forward, _native.stream_of(q)
        tables.use(stream)
        nbytes = plan.workspace
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        with _native.device_of(q):
            status = _native.library().ct_attention_forward(
                _operands(q, k, v, tables, causal, scale, rest), plan.entries, plan.counts, out.data_ptr(),
                _native.ptr(stats), _native.ptr(workspace), nbytes, stream)
        _native.check(status, "ct_attention_forward")
    return q, k, v, out, rest, stats


class _PackedAttention(torch.autograd.Function):
    """q [S, H, D], k and v [S_k, H_kv, D] on the device -> out [S, H, D]."""

    @staticmethod
    def forward(ctx, q, k, v, layout, causal, scale):
        q, k, v, out, rest, stats = _forward(q, k, v, layout, causal, scale, True)
        ctx.save_for_backward(q, k, v, out, rest, stats)
        ctx.layout, ctx.causal, ctx.scale = layout, causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, rest, stats = ctx.saved_tensors
        layout, causal, scale = ctx.layout, ctx.causal, ctx.scale
        _native.refuse_tangents("packed_attention", dout)
        if not layout.keys_disjoint:
            raise RuntimeError("packed_attention: key_records that overlap have no backward")
        tokens, heads, head_dim = q.shape
        key_tokens, kv_heads, _ = k.shape
        group, dtype, device = heads // kv_heads, q.dtype, q.device
        dout = _strided(dout, 64 // group + 2, group)
        work = layout.tokens and layout.key_tokens
        fresh = torch.empty if work and layout.whole and layout.tokens == tokens else torch.zeros
        dq = fresh((tokens, heads, head_dim), dtype=dtype, device=device)
        fresh = torch.empty if work and layout.keys_whole and layout.key_tokens == key_tokens else torch.zeros
        dk, dv = (fresh((key_tokens, kv_heads, head_dim), dtype=dtype, device=device) for _ in range(2))
        if work:
            tables = layout.tables(heads, kv_heads, head_dim, dtype, causal)
            rows, keys, stream = tables.rows, tables.keys, _native.stream_of(q)
            tables.use(stream)
            # the rows' terms, then the partial results of one pass after the other
            terms = -(-16 * tokens * heads // 256) * 256
            nbytes = max(rows.workspace, keys.workspace)
            scratch = torch.empty(max(terms + nbytes, 1), dtype=torch.uint8, device=device)
            at = scratch.data_ptr()
            dout_token, dout_head, _ = dout.stride()
            with _native.device_of(q):
                status = _native.library().ct_attention_backward(
                    _operands(q, k, v, tables, causal, scale, rest), rows.entries, rows.counts, keys.entries, keys.counts,
                    out.data_ptr(), stats.data_ptr(), dout.data_ptr(), dout_token, dout_head, at, dq.data_ptr(),
                    dk.data_ptr(), dv.data_ptr(), at + terms if nbytes else None, nbytes, stream)
            _native.check(status, "ct_attention_backward")
        return dq, dk, dv, None, None, None


def _host_attention(q, k, v, layout, causal, scale):
    """The same in torch operations, record by record in float32 (float64 for its tensors)."""
    group, wide = q.shape[1] // k.shape[1], torch.promote_types(q.dtype, torch.float32)
    out = q.new_zeros(q.shape)
    for (qa, qb), (ka, kb) in zip(layout.records, layout.key_records):
        if qa == qb or ka == kb:
            continue
        query = q[qa:qb].to(wide).transpose(0, 1)
        key, value = (t[ka:kb].to(wide).repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        s = (query @ key.transpose(1, 2)) * scale
        hidden = torch.zeros(qb - qa, kb - ka, dtype=torch.bool)
        if causal:
            hidden = torch.ones_like(hidden).triu((kb - ka) - (qb - qa) + 1)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        p = torch.where(hidden.all(-1)[:, None], torch.zeros_like(p), p)
        out = torch.cat((out[:qa], (p @ value).transpose(0, 1).to(q.dtype), out[qb:]))
    return out


def packed_attention(q, k, v, records, *, causal=True, scale=None):
    """softmax(scale q k^T) v inside each packed record; see the module docstring.

    q [S, H, D] or [1, S, H, D]; k and v [S_k, H_kv, D] (or [1, S_k, H_kv, D]) of the same
    dtype, H a multiple of H_kv, D a multiple of 8 up to 128, bf16 or float32 on the device, any
    strides (other than those of whole 16-byte pieces are copied first). `records` is an
    `AttentionLayout` or, for a single call, a list of (start, stop) spans. `scale` defaults to
    D ** -0.5. Returns a tensor of q's shape, differentiable in q, k and v
    (once, in reverse; host tensors in every way that torch offers)."""
    if q.dim() == 4 and q.shape[0] == 1 and k.dim() == 4 and k.shape[0] == 1 and v.dim() == 4 and v.shape[0] == 1:
        return packed_attention(q[0], k[0], v[0], records, causal=causal, scale=scale)[None]
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("packed_attention: q, k and v are [tokens, heads, head_dim] or [1, tokens, heads, head_dim]")
    if k.shape != v.shape:
        raise ValueError(f"packed_attention: keys {tuple(k.shape)} and values {tuple(v.shape)} differ")
    tokens, heads, head_dim = q.shape
    key_tokens, kv_heads, key_dim = k.shape
    if head_dim != key_dim or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"packed_attention: {heads} heads of {head_dim} do not share {kv_heads} of {key_dim}")
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError("packed_attention: mismatched element types")
    if not q.is_floating_point():
        raise ValueError("packed_attention: tensors of a floating type required")
    if not q.device == k.device == v.device:
        raise ValueError("packed_attention: q, k and v are on different devices")
    if head_dim == 0:
        raise ValueError("packed_attention: heads of no channels")
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:   # of float32's normal range, log2(e) times it too
        raise ValueError(f"packed_attention: scale {scale} is not a positive float32 number up to 2^126")
    layout = records if isinstance(records, AttentionLayout) else AttentionLayout(records, q.device)
    if layout.tokens > tokens or layout.key_tokens > key_tokens:
        raise ValueError(f"packed_attention: records reach to {layout.tokens} queries and {layout.key_tokens} keys, "
                         f"the tensors hold {tokens} and {key_tokens}")
    if layout.device != q.device:
        raise ValueError(f"packed_attention: the layout is on {layout.device}, the tensors on {q.device}")
    causal = bool(causal)
    if not q.is_cuda:
        return _host_attention(q, k, v, layout, causal, scale)
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("packed_attention: the HIP kernels take bfloat16 or float32")
    if head_dim % 8 or head_dim > 128:
        raise ValueError(f"packed_attention: head_dim {head_dim} is not a multiple of 8 up to 128")
    _native.refuse_tangents("packed_attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, layout, causal, scale)
    return _forward(q, k, v, layout, causal, scale, False)[3]
