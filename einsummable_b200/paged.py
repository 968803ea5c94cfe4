"""Descriptors of the paged key / value cache (es_paged_cache_t, es_cache_append_t, es_paged_attention_t of
the C ABI): what a step of generating tokens appends to and reads from.

The reference keeps one cache per layer and concatenates to it (attention_t::forward,
llama/modules.cc:285-383); here a layer's cache is a set of pages, a sequence a list of pages and a length.
kernel_manager_t.cache_append / paged_attention / prefix_attention and the program_t.add_* ops of the same
names take these descriptors with the arrays of a step.  A descriptor is built once and used every step.
"""
import ctypes

from . import _lib
from .scalarop import DTYPE_CODE

PAIRING_CODE = {"adjacent": 0, "halves": 1}


def _strides(c_array, values, name):
    values = [int(x) for x in values]
    if len(values) != len(c_array):
        raise ValueError("%s: expected %d strides" % (name, len(c_array)))
    for i, x in enumerate(values):
        c_array[i] = x


class paged_cache_t:
    """The cache of one layer and the batch of a step: `batch` sequences, `rows` rows in the step's tensors.
    k_stride / v_stride: elements between pages, tokens of a page and heads (the head dim is contiguous)."""

    def __init__(self, dtype, batch, rows, kv_heads, head_dim, page_size, n_pages, table_stride, k_stride, v_stride):
        c = _lib.es_paged_cache_t()
        c.dtype = DTYPE_CODE[dtype]
        c.batch, c.rows, c.kv_heads, c.head_dim = int(batch), int(rows), int(kv_heads), int(head_dim)
        c.page_size, c.n_pages, c.table_stride = int(page_size), int(n_pages), int(table_stride)
        _strides(c.k_stride, k_stride, "k_stride")
        _strides(c.v_stride, v_stride, "v_stride")
        self.c = c


class cache_append_t:
    """Rotated keys and values of the step's tokens into the cache, rotated queries out.  in_dtype: type of q, k
    and v (q_out has the cache's); heads: of the queries, 0 = none; strides: elements between rows and heads;
    rotary_dim 0 = no rotation; pairing "adjacent" (elements 2j, 2j + 1) or "halves" (j, j + rotary_dim / 2);
    n_positions: rows of the table of angles; pos_offset: added to every token's position."""

    def __init__(self, cache, in_dtype, heads, q_stride=(0, 0), k_stride=(0, 0), v_stride=(0, 0), q_out_stride=(0, 0),
                 n_positions=0, rotary_dim=0, pairing="adjacent", pos_offset=0):
        c = _lib.es_cache_append_t()
        c.cache = cache.c
        c.in_dtype, c.heads = DTYPE_CODE[in_dtype], int(heads)
        c.rotary_dim, c.pairing = int(rotary_dim), PAIRING_CODE[pairing]
        c.pos_offset, c.n_positions = int(pos_offset), int(n_positions)
        _strides(c.q_stride, q_stride, "q_stride")
        _strides(c.k_stride, k_stride, "k_stride")
        _strides(c.v_stride, v_stride, "v_stride")
        _strides(c.q_out_stride, q_out_stride, "q_out_stride")
        self.c = c
        self.ref = ctypes.byref(c)


class paged_attention_t:
    """Attention of the step's queries to their sequences' keys in the cache, each row up to its own token
    (causal) or to the whole sequence; prefix_len tokens shared by all sequences lie in front of them."""

    def __init__(self, cache, heads, scale, q_stride, out_stride, causal=True, prefix_len=0):
        c = _lib.es_paged_attention_t()
        c.cache = cache.c
        c.heads, c.causal, c.scale, c.prefix_len = int(heads), int(bool(causal)), float(scale), int(prefix_len)
        _strides(c.q_stride, q_stride, "q_stride")
        _strides(c.out_stride, out_stride, "out_stride")
        self.c = c
        self.ref = ctypes.byref(c)
