"""Appending to a paged cache and the attention that reads it, through the C ABI, against a plain restatement
in 64 bits (tests/paged_util.py, where the tolerances are derived)."""
import math

import pytest
import torch

import einsummable_b200 as es
from einsummable_b200 import program as es_program
from paged_util import TORCH, batch_t, check, truth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def km():
    return es.kernel_manager_t(0)


def cache_of(b):
    return es.paged_cache_t(b.dtype, b.batch, b.rows, b.kv_heads, b.dim, b.page, b.n_pages, b.tables.shape[1],
                            b.k_cache.stride()[:3], b.v_cache.stride()[:3])


def desc_of(b, causal=True):
    return es.paged_attention_t(cache_of(b), b.heads, b.scale, b.q.stride()[:2], b.out.stride()[:2], causal, b.prefix)


def attend(km, b, causal=True, lse=True, stream=None, desc=None, ws=None):
    desc = desc or desc_of(b, causal)
    if ws is None:
        n = km.paged_attention_workspace(desc)
        ws = (torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device=b.device), n)  # NaN in every word
    kw = dict(row_offsets=b.row_offsets, lse=b.lse if lse else None, workspace=ws)
    if b.prefix:
        km.prefix_attention(desc, stream, b.out, b.q, b.k_cache, b.v_cache, b.prefix_pages, b.lengths, b.tables, **kw)
    else:
        km.paged_attention(desc, stream, b.out, b.q, b.k_cache, b.v_cache, b.lengths, b.tables, **kw)


def run_and_check(km, b, causal=True):
    want = truth(b, causal)
    b.to(DEV)
    attend(km, b, causal)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    check(b, b.out, b.lse, want)


ONE = 1
ATTENTION = [
    # new, past, heads, kv_heads, dim, page, options
    ([1], [0], 1, 1, 128, 16, {}),                                   # the first token of all
    ([1], [-1], 4, 2, 64, 16, {}),                                   # a batch of one unused place
    ([1, 1, 1], [-1, 0, 200], 8, 2, 128, 16, {}),
    ([1], [1500], 32, 32, 128, 16, {}),                              # one row a key head, split along the keys
    ([1, 1], [63, 64], 8, 1, 64, 64, {}),                            # lengths of exactly one tile, and one more
    ([1] * 9, [0, 1, 14, 15, 16, 62, 126, 127, 700], 8, 8, 80, 7, {}),  # pages that end inside a tile
    ([1] * 3, [511, 512, 2000], 28, 4, 112, 48, {}),                 # 7 query heads a key head
    ([1], [900], 40, 1, 128, 32, {}),                                # 40 query heads on one key head
    ([1, 1], [300, 40], 64, 1, 96, 1, {}),                           # pages of one token
    ([1] * 300, [(37 * i) % 90 - 1 for i in range(300)], 4, 2, 32, 16, {}),  # more sequences than threads of a block
    ([1, 1], [700, 90], 12, 4, 128, 16, {"layout": "head"}),
    ([1, 1], [700, 90], 12, 4, 100, 16, {"layout": "odd"}),          # nothing aligned
    ([1], [300], 4, 2, 256, 16, {}),
    ([1, 1], [300, 5], 3, 3, 1, 16, {}),
    ([1, 1], [600, 33], 16, 4, 64, 16, {"dtype": "f32"}),
    ([1], [2500], 8, 1, 128, 16, {"dtype": "f32"}),
    ([1], [129], 2, 2, 250, 16, {"dtype": "f32"}),
    ([1, 1], [129, 7], 6, 2, 100, 16, {"dtype": "f32", "layout": "odd"}),
    # several rows a sequence
    ([5], [0], 4, 4, 128, 16, {}),
    ([3, 0, 1, 130, 17], [5, 9, 0, 70, 1000], 8, 2, 128, 16, {"spare": 3}),
    ([40, 2], [0, 333], 28, 4, 64, 24, {}),
    ([300], [41], 8, 1, 128, 64, {}),
    ([4, 6], [-2, -6], 4, 2, 64, 16, {}),                            # rows in front of the first token see nothing
    ([0, 0], [5, 0], 4, 2, 64, 16, {"spare": 4}),                    # no row at all
    ([65, 33, 1], [0, 500, 64], 4, 4, 80, 16, {}),
    ([20, 3], [11, 200], 6, 2, 48, 16, {"dtype": "f32", "spare": 2}),
    ([9, 30], [11, 200], 6, 2, 30, 16, {"layout": "odd"}),
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,opt", ATTENTION)
def test_paged_attention(km, new, past, heads, kv_heads, dim, page, opt):
    run_and_check(km, batch_t(new, past, heads, kv_heads, dim, page, seed=len(new) + dim, **opt))


@pytest.mark.parametrize("new,past", [([1, 1, 1], [7, 400, -1]), ([3, 70], [150, 12])])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_not_causal(km, new, past, dtype):
    """Every row sees the whole sequence, as queries on an encoder's states do."""
    run_and_check(km, batch_t(new, past, 8, 4, 64, 16, dtype=dtype, seed=3), causal=False)


PREFIX = [
    ([1], [0], 4, 4, 128, 16, 1, {}),
    ([1, 1, 1], [0, 40, -1], 8, 2, 128, 16, 500, {}),          # an unused place sees the prefix only
    ([1] * 70, [i % 33 for i in range(70)], 8, 2, 128, 16, 1000, {}),
    ([1] * 40, [i for i in range(40)], 4, 4, 64, 48, 129, {}),
    ([1] * 5, [3, 0, 17, 90, 300], 28, 4, 112, 16, 64, {}),
    ([2, 0, 9, 1], [0, 4, 30, 7], 8, 4, 80, 7, 200, {"spare": 2}),
    ([1] * 6, [3, 0, 17, 90, 300, 2], 8, 4, 64, 16, 333, {"dtype": "f32"}),
    ([1] * 6, [3, 0, 17, 90, 300, 2], 8, 4, 100, 16, 333, {"layout": "odd"}),
    ([1] * 130, [i % 5 for i in range(130)], 2, 1, 128, 64, 4000, {}),
    # the prefix read once for few rows, on the tensor cores and without
    ([1] * 3, [0, 31, -1], 32, 8, 128, 16, 6000, {}),
    ([1] * 4, [5, 0, 70, -1], 8, 4, 64, 16, 500, {"offsets": True}),
    ([1] * 4, [5, 0, 70, -1], 8, 4, 64, 16, 500, {"offsets": True, "dtype": "f32"}),
    ([1] * 4, [5, 0, 70, 260], 8, 4, 64, 16, 15, {}),               # a prefix that ends inside a key tile
    ([1] * 9, [5, 0, 70, 260, 1, 2, 3, 4, 5], 8, 4, 64, 24, 100, {}),
    ([1] * 40, [i for i in range(40)], 32, 1, 128, 16, 200, {"offsets": True}),  # 32 heads on one key head: 1280 rows
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,prefix,opt", PREFIX)
def test_prefix_attention(km, new, past, heads, kv_heads, dim, page, prefix, opt):
    run_and_check(km, batch_t(new, past, heads, kv_heads, dim, page, prefix=prefix, seed=len(new) + dim, **opt))


def test_prefix_of_no_tokens_is_paged_attention(km):
    b = batch_t([1, 1], [40, 600], 8, 2, 128, 16, seed=5).to(DEV)
    attend(km, b)
    want = b.out.clone()
    b.out.zero_()
    desc = desc_of(b)
    n = km.paged_attention_workspace(desc)
    km.prefix_attention(desc, None, b.out, b.q, b.k_cache, b.v_cache, None, b.lengths, b.tables,
                        workspace=(torch.empty(max(n, 16), dtype=torch.uint8, device=DEV), n))
    torch.cuda.synchronize()
    assert torch.equal(b.out, want)


def test_the_same_bits_every_time(km):
    b = batch_t([1] * 5, [3000, 10, 700, 64, 1999], 8, 2, 128, 16, seed=6).to(DEV)
    attend(km, b)
    first, lse = b.out.clone(), b.lse.clone()
    for _ in range(5):
        attend(km, b)
        assert torch.equal(b.out, first) and torch.equal(b.lse, lse)


def test_without_lse_and_far_scores(km):
    """Scores of several hundred: only the differences from the maximum count."""
    b = batch_t([1, 1], [90, 700], 8, 2, 64, 16, seed=7)
    b.q *= 60
    want = truth(b)
    b.to(DEV)
    attend(km, b, lse=False)
    check(b, b.out, None, want)
    assert (b.lse == 7).all()


# ------------------------------------------------------------------------------------------- append
def append_inputs(b, in_dtype, rotary_dim, seed, packed=True):
    g = torch.Generator().manual_seed(seed)
    dt = TORCH[in_dtype]
    x = torch.randn((b.rows, b.heads + 2 * b.kv_heads, b.dim), generator=g).to(dt)
    q, k, v = x.split([b.heads, b.kv_heads, b.kv_heads], 1)
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    n = max(max(b.total), 1) + 40
    ang = torch.arange(n).double().unsqueeze(1) * 10000.0 ** (-torch.arange(0, max(rotary_dim, 2), 2).double() / max(rotary_dim, 2))
    freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    return q, k, v, freqs


def turned(x, f, rotary_dim, halves):
    """x [heads, dim] in 64 bits, f [rotary_dim / 2] complex128."""
    y = x.clone()
    h = rotary_dim // 2
    a, b = (x[:, :h], x[:, h:rotary_dim]) if halves else (x[:, 0:rotary_dim:2], x[:, 1:rotary_dim:2])
    re, im = a * f.real - b * f.imag, a * f.imag + b * f.real
    if halves:
        y[:, :h], y[:, h:rotary_dim] = re, im
    else:
        y[:, 0:rotary_dim:2], y[:, 1:rotary_dim:2] = re, im
    return y


APPEND = [
    # new, past, heads, kv_heads, dim, page, in, cache, rotary, pairing, options
    ([1], [0], 4, 2, 128, 16, "f16", "f16", 128, "adjacent", {}),
    ([1], [700], 32, 8, 128, 16, "f16", "f16", 128, "halves", {}),
    ([1] * 300, [i % 40 - 1 for i in range(300)], 8, 2, 64, 16, "f16", "f16", 64, "adjacent", {"offsets": True}),
    ([3, 0, 1, 130, 17], [5, 9, 0, 70, 100], 8, 2, 128, 16, "f16", "f16", 128, "adjacent", {"spare": 3}),
    ([4, 6], [-2, -6], 4, 2, 80, 16, "f16", "f16", 80, "halves", {}),     # rows without a place
    ([20, 2], [0, 30], 4, 4, 112, 7, "f32", "f16", 64, "adjacent", {}),   # part of a head rotated
    ([20, 2], [0, 30], 4, 4, 112, 7, "f32", "f16", 64, "halves", {}),
    ([20, 2], [0, 30], 6, 2, 64, 24, "f32", "f32", 64, "halves", {}),
    ([20, 2], [0, 30], 6, 2, 64, 24, "f16", "f32", 0, "adjacent", {}),    # no rotation
    ([5, 2], [0, 30], 3, 1, 30, 5, "f16", "f16", 30, "adjacent", {"layout": "odd"}),
    ([5, 2], [0, 30], 3, 1, 30, 5, "f32", "f16", 22, "halves", {"layout": "odd"}),
    ([5, 2], [0, 30], 3, 1, 37, 5, "f16", "f16", 36, "halves", {"layout": "odd"}),
    ([5, 2], [0, 30], 3, 1, 256, 5, "f16", "f16", 12, "adjacent", {"layout": "head"}),
    ([5, 2], [0, 30], 0, 2, 64, 5, "f16", "f16", 64, "adjacent", {}),     # no queries
    ([1, 1], [9, 3], 2, 1, 1, 4, "f16", "f16", 0, "adjacent", {}),
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,tin,tc,rot,pairing,opt", APPEND)
def test_cache_append(km, new, past, heads, kv_heads, dim, page, tin, tc, rot, pairing, opt):
    b = batch_t(new, past, max(heads, kv_heads), kv_heads, dim, page, dtype=tc, seed=dim, filler=0.25, **opt)
    b.heads = heads
    q, k, v, freqs = append_inputs(b, tin, rot, seed=1)
    pos_offset = 13
    q_out = torch.full((b.rows, max(heads, 1), dim), 3.0, dtype=TORCH[tc])
    wq, wk, wv = q_out.double(), b.k_cache.double(), b.v_cache.double()
    tq, tk, tv = torch.zeros_like(wq), torch.zeros_like(wk), torch.zeros_like(wv)
    f64 = freqs.to(torch.complex128)
    u = 2.0 ** -11 if tc == "f16" else 2.0 ** -24

    def bound(x, y):  # two products and a sum in f32 (3 roundings of 2^-24 of |x c| + |y s|), then one to the type
        return u * y.abs() * (1 + 2.0 ** -8) + 3 * 2.0 ** -24 * 2 * x.abs().max() + 2.0 ** -25

    for i in range(b.batch):
        for r in range(new[i]):
            p = b.total[i] - new[i] + r
            if p < 0:
                continue
            row, f = b.off[i] + r, f64[p + pos_offset]
            at = (b.tables[i, p // page].long(), p % page)
            if heads:
                wq[row] = turned(q[row].double(), f, rot, pairing == "halves")
                tq[row] = bound(q[row].double(), wq[row])
            wk[at] = turned(k[row].double(), f, rot, pairing == "halves")
            tk[at] = bound(k[row].double(), wk[at])
            wv[at] = v[row].double()
            # half a step of f16 is 2^-11 of the value, and 2^-25 for values below 2^-14 (steps of 2^-24)
            tv[at] = u * wv[at].abs() + 2.0 ** -25 if tin == "f32" and tc == "f16" else 0.0
    b.to(DEV)
    dev = [t.to(DEV) for t in (q, k, v)] if opt.get("layout") else list(torch.cat([q, k, v], 1).to(DEV).split(
        [heads, kv_heads, kv_heads], 1))
    q_out, freqs = q_out.to(DEV), freqs.to(DEV)
    d = es.cache_append_t(cache_of(b), tin, heads, dev[0].stride()[:2], dev[1].stride()[:2], dev[2].stride()[:2],
                          q_out.stride()[:2], freqs.shape[0], rot, pairing, pos_offset)
    km.cache_append(d, None, b.k_cache, b.v_cache, dev[1], dev[2], b.lengths, b.tables, b.row_offsets, freqs if rot else None,
                    dev[0] if heads else None, q_out if heads else None)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    for got, want, tol in ((q_out, wq, tq), (b.k_cache, wk, tk), (b.v_cache, wv, tv)):
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), ((err - tol).max().item(), (err > tol).sum().item())


def test_append_in_place(km):
    """The queries rotated where they are."""
    b = batch_t([3, 1], [2, 40], 8, 2, 128, 16, seed=2, filler=0.25)
    q, k, v, freqs = append_inputs(b, "f16", 128, seed=4, packed=False)
    b.to(DEV)
    q, k, v, freqs = (t.to(DEV) for t in (q, k, v, freqs))
    outs = []
    for inplace in (False, True):
        qi = q.clone()
        qo = qi if inplace else torch.empty_like(qi)
        d = es.cache_append_t(cache_of(b), "f16", 8, qi.stride()[:2], k.stride()[:2], v.stride()[:2], qo.stride()[:2],
                              freqs.shape[0], 128, "halves")
        km.cache_append(d, None, b.k_cache, b.v_cache, k, v, b.lengths, b.tables, b.row_offsets, freqs, qi, qo)
        outs.append(qo)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
