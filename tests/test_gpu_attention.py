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


@pytest.mark.parametrize("dtype,length,heads,kv_heads,dim", [
    (torch.bfloat16, 1500, 4, 1, 128), (torch.bfloat16, 1111, 4, 4, 64), (torch.float32, 700, 3, 1, 128)])
def test_long_records(dtype, length, heads, kv_heads, dim):
    """Long enough that every pass runs many tiles and the key gradients are joined from parts."""
    _case([length, 300], [length, 300], heads, kv_heads, dim, dtype, True)
