"""The paged-cache operators without a GPU: what they refuse, the workspace they ask for, their place in a
program's schedule, and the plain restatement that the GPU tests compare with."""
import math

import pytest
import torch

import einsummable_b200 as es
from einsummable_b200 import _lib
from einsummable_b200.program import program_t
from paged_util import batch_t, truth

PTR = 1 << 20  # a device address that nothing here reads


def cache(dtype="f16", batch=2, rows=2, kv_heads=2, head_dim=64, page_size=16, n_pages=8, table_stride=4, k_stride=None, v_stride=None):
    st = (page_size * kv_heads * head_dim, kv_heads * head_dim, head_dim)
    return es.paged_cache_t(dtype, batch, rows, kv_heads, head_dim, page_size, n_pages, table_stride, k_stride or st, v_stride or st)


def attention(c=None, heads=4, scale=0.125, q_stride=(256, 64), out_stride=(256, 64), causal=True, prefix_len=0):
    return es.paged_attention_t(c or cache(), heads, scale, q_stride, out_stride, causal, prefix_len)


def add_attention(desc, **kw):
    p = program_t(None)
    a = dict(out=PTR, q=PTR, k_cache=PTR, v_cache=PTR, lengths=PTR, tables=PTR)
    a.update(kw)
    p.add_paged_attention(desc, **a)
    return p


def append(c=None, in_dtype="f16", heads=4, n_positions=100, rotary_dim=64, pairing="adjacent", pos_offset=0, **strides):
    s = dict(q_stride=(256, 64), k_stride=(128, 64), v_stride=(128, 64), q_out_stride=(256, 64))
    s.update(strides)
    return es.cache_append_t(c or cache(), in_dtype, heads, n_positions=n_positions, rotary_dim=rotary_dim, pairing=pairing,
                             pos_offset=pos_offset, **s)


def add_append(desc, **kw):
    p = program_t(None)
    a = dict(k_cache=PTR, v_cache=PTR, k=PTR, v=PTR, lengths=PTR, tables=PTR, freqs=PTR, q=PTR, q_out=PTR)
    a.update(kw)
    p.add_cache_append(desc, **a)
    return p


@pytest.mark.parametrize("make,status", [
    (lambda: attention(cache(dtype="f64")), _lib.ES_NOT_SUPPORTED),
    (lambda: attention(cache(dtype="c64")), _lib.ES_NOT_SUPPORTED),
    (lambda: attention(cache(head_dim=257)), _lib.ES_NOT_SUPPORTED),
    (lambda: attention(cache(head_dim=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(batch=0, rows=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(page_size=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(n_pages=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(table_stride=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(kv_heads=0)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(cache(rows=3)), _lib.ES_BAD_DESCRIPTOR),               # without row offsets: a row a sequence
    (lambda: attention(cache(k_stride=(-1, 128, 64))), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(heads=3), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(heads=0), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(scale=0.0), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(scale=-1.0), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(scale=math.inf), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(scale=math.nan), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(q_stride=(256, -64)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: attention(prefix_len=10), _lib.ES_BAD_ARGUMENT),                 # and no list of its pages
    (lambda: attention(prefix_len=(1 << 30) + 1), _lib.ES_NOT_SUPPORTED),
])
def test_attention_refuses_descriptors(make, status):
    with pytest.raises(es.es_error) as e:
        add_attention(make())
    assert e.value.status == status


@pytest.mark.parametrize("kw", [{k: None} for k in ("out", "q", "k_cache", "v_cache", "lengths", "tables")] + [
    {"q": PTR + 1}, {"out": PTR + 1}, {"k_cache": PTR + 1}, {"lengths": PTR + 2}, {"tables": PTR + 2}, {"lse": PTR + 2},
    {"row_offsets": PTR + 2}])
def test_attention_refuses_pointers(kw):
    with pytest.raises(es.es_error) as e:
        add_attention(attention(), **kw)
    assert e.value.status == _lib.ES_BAD_ARGUMENT


@pytest.mark.parametrize("make,status", [
    (lambda: append(cache(dtype="f64")), _lib.ES_NOT_SUPPORTED),
    (lambda: append(in_dtype="f64"), _lib.ES_NOT_SUPPORTED),
    (lambda: append(rotary_dim=63), _lib.ES_BAD_DESCRIPTOR),
    (lambda: append(rotary_dim=66), _lib.ES_BAD_DESCRIPTOR),
    (lambda: append(n_positions=0), _lib.ES_BAD_ARGUMENT),
    (lambda: append(pos_offset=-1), _lib.ES_BAD_DESCRIPTOR),
    (lambda: append(heads=70000), _lib.ES_NOT_SUPPORTED),
    (lambda: append(cache(rows=5)), _lib.ES_BAD_DESCRIPTOR),
    (lambda: append(k_stride=(-128, 64)), _lib.ES_BAD_DESCRIPTOR),
])
def test_append_refuses_descriptors(make, status):
    with pytest.raises(es.es_error) as e:
        add_append(make())
    assert e.value.status == status


@pytest.mark.parametrize("kw", [{k: None} for k in ("k_cache", "v_cache", "k", "v", "lengths", "tables", "freqs", "q", "q_out")] + [
    {"k": PTR + 1}, {"q_out": PTR + 1}, {"freqs": PTR + 2}, {"tables": PTR + 1}])
def test_append_refuses_pointers(kw):
    with pytest.raises(es.es_error) as e:
        add_append(append(), **kw)
    assert e.value.status == _lib.ES_BAD_ARGUMENT


def test_append_without_queries_or_rotation_needs_neither():
    add_append(append(heads=0, rotary_dim=0, n_positions=0), q=None, q_out=None, freqs=None)


def test_unknown_pairing_and_wrong_stride_counts():
    with pytest.raises(KeyError):
        append(pairing="quarters")
    with pytest.raises(ValueError):
        attention(q_stride=(1, 2, 3))
    with pytest.raises(ValueError):
        cache(k_stride=(1, 2))


def workspace(desc):
    import ctypes
    n = ctypes.c_uint64(0)
    _lib.check(_lib.load().es_b200_paged_attention_workspace(ctypes.byref(desc.c), ctypes.byref(n)))
    return n.value


def test_workspace_does_not_grow_with_the_lengths():
    """It depends on the machine's width, and with a prefix on the rows -- not on how many keys there are."""
    short, long = attention(cache(table_stride=1)), attention(cache(table_stride=100000, n_pages=1 << 20))
    assert workspace(short) == workspace(long) > 0
    with_prefix = attention(prefix_len=1000)
    assert workspace(with_prefix) - workspace(short) == 2 * 4 * 64 * 4 + 256  # rows x heads x dim f32, and the lse, each 256-aligned
    assert workspace(attention(cache(dtype="f32"))) <= workspace(short)


def test_a_step_as_ops_of_a_program():
    """append -> attention: two ops in order, and the attention's workspace is part of the program's."""
    p = program_t(None)
    a = p.add_cache_append(append(), PTR, PTR, PTR, PTR, PTR, PTR, freqs=PTR, q=PTR, q_out=PTR)
    b = p.add_paged_attention(attention(), PTR, PTR, PTR, PTR, PTR, PTR, deps=[a])
    ws = p.finalize()
    assert ws >= workspace(attention())
    ops = p.describe()["ops"]
    assert [o["kind"] for o in ops] == ["cache_append", "paged_attention"]
    assert ops[b]["lane"] == ops[a]["lane"]


def test_restatement_against_a_dense_softmax():
    """The 64-bit restatement on one sequence is softmax(scale q k^T + mask) v over the gathered keys."""
    b = batch_t([4], [9], 6, 2, 8, 5, dtype="f32", seed=3)
    out, lse, tol, _ = truth(b)
    keys = torch.stack([b.k_cache[b.tables[0, p // 5].long(), p % 5] for p in range(13)]).double()
    vals = torch.stack([b.v_cache[b.tables[0, p // 5].long(), p % 5] for p in range(13)]).double()
    for r in range(4):
        for h in range(6):
            s = (keys[:, h // 3] @ b.q[r, h].double()) * b.scale
            s[9 + r + 1:] = -math.inf
            w = torch.softmax(s, 0) @ vals[:, h // 3]
            assert (out[r, h] - w).abs().max() < 1e-12
            assert abs(lse[r, h] - torch.logsumexp(s, 0)) < 1e-12
    assert (tol > 0).all()
