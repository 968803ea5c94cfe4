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
    ([1, 1], [1900, 20], 32, 2, 128, 16, {}),                        # 16
    ([1, 1], [1900, 20], 34, 2, 64, 16, {}),                         # 17
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


@pytest.mark.parametrize("past,heads,kv_heads,dim,page,prefix", [
    # no tile, one, as many as the block has warps, one more, ... up to the longest that a block takes
    ([-1, 0, 15, 16, 46, 47, 63, 64, 65, 1023], 32, 8, 128, 16, 0),
    ([-1, 0, 15, 16, 46, 47, 63, 64, 65, 700], 14, 2, 80, 7, 0),
    ([1023, 5], 16, 1, 64, 64, 0),
    ([300, 0, -1], 80, 2, 128, 16, 0),
    ([300, 0, -1], 16, 4, 128, 16, 37),                          # a prefix in front of each
    ([17, 0, -1, 500], 16, 4, 64, 16, 40000),                    # one that is joined in
])
def test_a_block_a_sequence_and_key_head(km, past, heads, kv_heads, dim, page, prefix):
    run_and_check(km, batch_t([1] * len(past), past, heads, kv_heads, dim, page, prefix=prefix, seed=dim + prefix))


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
    ([1] * 70, [i % 33 for i in range(70)], 8, 2, 128, 16, 4000, {}),            # read once, 280 rows a key head
    ([1] * 4, [3, 0, 17, -1], 8, 2, 128, 16, 3500, {"offsets": True}),           # 16 rows
    ([1] * 5, [3, 0, 17, -1, 40], 8, 2, 64, 24, 900, {"offsets": True}),         # 20
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


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("new,prefix", [(1, 0), (60, 0), (1, 40), (3, 40), (60, 40)])
def test_values_that_are_not_finite_stay_in_their_rows(km, dtype, new, prefix):
    """NaN in a query spoils that row's head, NaN in a key or infinities in a value that sequence's rows, and
    nothing else -- not the memory behind a result that is not there, either."""
    b = batch_t([new] * 4, [40, 200, 90, 33], 8, 2, 64, 16, dtype=dtype, prefix=prefix, seed=17)
    want = truth(b)
    b.q[b.off[0], 5] = float("nan")
    b.k_cache[b.tables[1, 0].long(), 3, 1] = float("nan")  # key head 1: query heads 4 .. 7
    b.v_cache[b.tables[2, 1].long(), 2, 0] = float("inf")  # key head 0
    b.to(DEV)
    attend(km, b)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    out, lse = b.out.cpu().double(), b.lse.cpu().double()
    spoiled = torch.zeros(b.rows, 8, dtype=torch.bool)
    spoiled[b.off[0], 5] = True
    spoiled[b.off[1]:b.off[2], 4:] = True
    spoiled[b.off[2]:b.off[3], :4] = True
    assert torch.isnan(out[b.off[0], 5]).all() and torch.isnan(lse[b.off[0], 5])
    assert torch.isnan(out[b.off[1]:b.off[2], 4:]).all() and torch.isnan(lse[b.off[1]:b.off[2], 4:]).all()
    assert not torch.isfinite(out[b.off[2]:b.off[3], :4]).any()
    clean = ~spoiled
    assert ((out - want[0]).abs() <= want[2])[clean].all()
    assert ((lse - want[1]).abs() <= want[3])[clean].all()


# --------------------------------------------------------------------------------- what the arrays hold
def status_after(km, b, **kw):
    attend(km, b, **kw)
    torch.cuda.synchronize()
    first = km.device_status()
    assert km.device_status() == 0  # reading it clears it
    return first


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("new", [1, 50])
def test_a_page_that_does_not_exist_spoils_its_own_sequence_only(km, dtype, page, new):
    b = batch_t([new, 1, new], [40, 200, 90], 8, 2, 64, page, dtype=dtype, seed=9)
    want = truth(b)
    b.to(DEV)
    b.tables[1, 3] = b.n_pages
    assert status_after(km, b) == 0x21
    b.tables[1, 3] = -5
    assert status_after(km, b) == 0x21
    keep = torch.ones(b.rows, dtype=torch.bool)
    keep[b.off[1]:b.off[2]] = False
    got, lse = b.out.cpu()[keep], b.lse.cpu()[keep]
    assert ((got.double() - want[0][keep]).abs() <= want[2][keep]).all()
    assert ((lse.double() - want[1][keep]).abs() <= want[3][keep]).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lengths_that_the_tables_cannot_hold(km, dtype):
    b = batch_t([1, 1, 1], [40, 200, 90], 8, 2, 64, 16, dtype=dtype, seed=9)
    want = truth(b)
    b.to(DEV)
    for bad in (b.tables.shape[1] * 16 + 1, -1, 2 ** 31 - 1, -2 ** 31):
        b.lengths[1] = bad
        assert status_after(km, b) == 0x22
        assert (b.out[1] == 0).all() and torch.isinf(b.lse[1]).all()  # as a sequence without keys
        for i in (0, 2):
            assert ((b.out[i].cpu().double() - want[0][i]).abs() <= want[2][i]).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_row_offsets_that_fall_or_pass_the_rows(km, dtype):
    for off in ([0, 3, 2, 5], [0, 2, 5, 99], [-1, 2, 3, 5], [0, 2, 2 ** 31 - 1, 5]):
        b = batch_t([2, 1, 2], [40, 200, 90], 8, 2, 64, 16, dtype=dtype, seed=9).to(DEV)
        b.row_offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
        assert status_after(km, b) == 0x23
        b = batch_t([2, 1, 2], [40, 200, 90], 8, 2, 64, 16, dtype=dtype, seed=9, prefix=70).to(DEV)
        b.row_offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
        assert status_after(km, b) == 0x23


def append_desc(b, dev, q_out, n, **kw):
    return es.cache_append_t(cache_of(b), b.dtype, b.heads, dev[0].stride()[:2], dev[1].stride()[:2], dev[2].stride()[:2],
                             q_out.stride()[:2], n, b.dim, **kw)


@pytest.mark.parametrize("spoil,code", [("page", 0x21), ("length", 0x22), ("offsets", 0x23), ("position", 0x24)])
def test_append_with_bad_arrays(km, spoil, code):
    """Nothing of the bad sequence is written, everything of the others is."""
    def run(bad):
        b = batch_t([2, 3, 1], [5, 40, 17], 4, 2, 64, 16, seed=4, filler=0.5)
        q, k, v, freqs = append_inputs(b, "f16", 64, seed=8)
        b.to(DEV)
        dev, n = [t.contiguous().to(DEV) for t in (q, k, v)], freqs.shape[0]
        q_out = torch.full_like(dev[0], 3.0)
        if bad == "page":
            b.tables[1, 2] = 1 << 28
        elif bad == "length":
            b.lengths[1] = 1 << 28
        elif bad == "offsets":
            b.row_offsets[2] = 1 << 28
        elif bad == "position":
            n = 30  # positions 40 .. 42 lie behind the table's end
        km.cache_append(append_desc(b, dev, q_out, n), None, b.k_cache, b.v_cache, dev[1], dev[2], b.lengths, b.tables, b.row_offsets,
                        freqs.to(DEV), dev[0], q_out)
        torch.cuda.synchronize()
        return b, q_out, km.device_status()

    good, q_good, status = run(None)
    assert status == 0
    b, q_out, status = run(spoil)
    assert status == code
    owned = [(good.tables[i, p // 16].long().item(), p % 16) for i in (0, 2) for p in range(good.total[i])]
    if spoil == "offsets":  # the last sequence begins where the bad one claims to end
        owned = owned[:good.total[0]]
    for pg, sl in owned:
        assert torch.equal(b.k_cache[pg, sl], good.k_cache[pg, sl]) and torch.equal(b.v_cache[pg, sl], good.v_cache[pg, sl])
    assert torch.equal(q_out[:2], q_good[:2])
    before = batch_t([2, 3, 1], [5, 40, 17], 4, 2, 64, 16, seed=4, filler=0.5)
    for p in range(40, 43):
        pg, sl = before.tables[1, p // 16].long().item(), p % 16
        assert torch.equal(b.k_cache[pg, sl].cpu(), before.k_cache[pg, sl]), "a row without a place was written"


def test_workspace_is_checked(km):
    b = batch_t([1], [100], 4, 2, 64, 16, seed=1).to(DEV)
    n = km.paged_attention_workspace(desc_of(b))
    small = torch.empty(n - 1, dtype=torch.uint8, device=DEV)
    for ws in (None, (small, n - 1)):
        with pytest.raises(es.es_error) as e:
            km.paged_attention(desc_of(b), None, b.out, b.q, b.k_cache, b.v_cache, b.lengths, b.tables, workspace=ws)
        assert e.value.status == 3
    with pytest.raises(es.es_error) as e:
        off = torch.empty(n + 64, dtype=torch.uint8, device=DEV)
        km.paged_attention(desc_of(b), None, b.out, b.q, b.k_cache, b.v_cache, b.lengths, b.tables, workspace=(off[1:], n))
    assert e.value.status == 6


# -------------------------------------------------------------------------------------- in real use
def test_sequences_that_share_pages(km):
    """Two continuations of one text hold the same pages in front, and different ones behind."""
    b = batch_t([1, 1], [99, 120], 8, 2, 128, 16, seed=11)
    b.tables[1, :4] = b.tables[0, :4]
    want = truth(b)
    b.to(DEV)
    attend(km, b)
    torch.cuda.synchronize()
    check(b, b.out, b.lse, want)


def test_offsets_beyond_32_bits(km):
    """Pages whose elements lie beyond 2^32: 300000 pages of 16 tokens, 8 heads of 128 (9.8 GB)."""
    g = torch.Generator(device=DEV).manual_seed(3)
    pool = torch.empty((300000, 16, 8, 128), dtype=torch.float16, device=DEV)
    for new, past in (([1, 1], [100, 700]), ([70, 1], [40, 90])):
        b = batch_t(new, past, 16, 8, 128, 16, seed=12)
        far = torch.randperm(30000, generator=torch.Generator().manual_seed(1))[:b.n_pages] + 270000
        held = b.tables < b.n_pages
        pool[far.to(DEV)] = torch.randn((b.n_pages, 16, 8, 128), generator=g, device=DEV, dtype=torch.float16)
        b.k_cache = b.v_cache = pool[far.to(DEV)].cpu()
        want = truth(b)
        b.tables = torch.where(held, far[b.tables.clamp(0, b.n_pages - 1).long()].to(torch.int32), b.tables)
        b.to(DEV)
        b.k_cache = b.v_cache = pool
        b.n_pages = 300000
        attend(km, b)
        torch.cuda.synchronize()
        assert km.device_status() == 0
        check(b, b.out, b.lse, want)
        # and written there
        x = torch.randn((b.rows, 8, 128), generator=g, device=DEV, dtype=torch.float16)
        d = es.cache_append_t(cache_of(b), "f16", 0, k_stride=x.stride()[:2], v_stride=x.stride()[:2])
        km.cache_append(d, None, pool, pool, x, x, b.lengths, b.tables, b.row_offsets)
        torch.cuda.synchronize()
        last = b.total[1] - 1
        assert torch.equal(pool[b.tables[1, last // 16].long(), last % 16], x[-1])


def test_two_streams_with_a_workspace_each(km):
    """Calls that overlap in time, each on a stream and with a workspace of its own."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    made = []
    for i, (new, past, prefix) in enumerate([([1] * 9, [700 + 31 * k for k in range(9)], 0), ([90, 40], [300, 5], 0),
                                             ([1] * 70, [k % 9 for k in range(70)], 1500)]):
        b = batch_t(new, past, 8, 2, 128, 16, prefix=prefix, seed=20 + i)
        want = truth(b)
        b.to(DEV)
        n = km.paged_attention_workspace(desc_of(b))
        made.append((b, want, desc_of(b), (torch.empty(n, dtype=torch.uint8, device=DEV), n)))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (b, _, d, ws) in zip(streams, made):
            attend(km, b, stream=s, desc=d, ws=ws)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    for b, want, _, _ in made:
        check(b, b.out, b.lse, want)


def test_captured_calls_share_a_workspace_and_follow_the_lengths(km):
    """Two captured calls with one workspace between them, replayed in turn after the lengths on the device changed."""
    made, graphs = [], []
    n = 0
    for i, (heads, kv) in enumerate([(8, 2), (40, 1)]):
        b = batch_t([1, 1, 1], [1000, 300, 44], heads, kv, 128, 16, seed=30 + i)
        host = batch_t([1, 1, 1], [1000, 300, 44], heads, kv, 128, 16, seed=30 + i)
        made.append((b.to(DEV), host))
        n = max(n, km.paged_attention_workspace(desc_of(b)))
    ws = (torch.empty(n, dtype=torch.uint8, device=DEV), n)
    s = torch.cuda.Stream()
    for b, _ in made:
        attend(km, b, stream=s, ws=ws)  # once before the capture: everything is loaded
    torch.cuda.synchronize()
    for b, _ in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attend(km, b, stream=torch.cuda.current_stream(), ws=ws)
        graphs.append(g)
    for shorter in (0, 17, 43):
        for b, host in made:
            b.lengths.copy_(host.lengths.to(DEV) - shorter)
            b.out.fill_(9)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for _ in range(2):
                for g in graphs:
                    g.replay()
        torch.cuda.synchronize()
        for b, host in made:
            host.total = [t - shorter for t in (1001, 301, 45)]
            check(b, b.out, b.lse, truth(host))
    del graphs


@pytest.mark.parametrize("prefix", [0, 70, 5000])
def test_generating_with_a_program(km, prefix):
    """Prompts of different lengths, then tokens one by one: append and attention as two ops of a program, the
    step captured once and replayed with the lengths, rows and pages changed on the device -- against the dense
    softmax over everything that was appended so far.  The keys come back from the cache rotated."""
    heads, kv, dim, page, steps = 8, 2, 64, 16, 6
    prompts = [5, 33, 1]
    g = torch.Generator().manual_seed(7)
    width = 5
    n_prefix = -(-prefix // page)
    n_pages = 3 * width + n_prefix + 1
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    tables = order[:3 * width].view(3, width).contiguous().to(DEV)
    shared = order[3 * width:3 * width + n_prefix].contiguous().to(DEV)
    k_cache = torch.zeros((n_pages, page, kv, dim), dtype=torch.float16, device=DEV)
    v_cache = torch.zeros_like(k_cache)
    ang = torch.arange(prefix + 100).double().unsqueeze(1) * 10000.0 ** (-torch.arange(0, dim, 2).double() / dim)
    freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    dfreqs = freqs.to(DEV)
    if prefix:
        pk = torch.randn((prefix, kv, dim), generator=g).half()
        pv = torch.randn((prefix, kv, dim), generator=g).half()
        at = torch.arange(prefix)
        k_cache[shared.cpu().long()[at // page].to(DEV), (at % page).to(DEV)] = pk.to(DEV)
        v_cache[shared.cpu().long()[at // page].to(DEV), (at % page).to(DEV)] = pv.to(DEV)
    keys = [[] for _ in prompts]   # rotated, as they were rounded into the cache
    vals = [[] for _ in prompts]
    lengths = torch.zeros(3, dtype=torch.int32, device=DEV)

    def plan(rows, offsets):
        c = es.paged_cache_t("f16", 3, rows, kv, dim, page, n_pages, width, k_cache.stride()[:3], v_cache.stride()[:3])
        x = torch.empty((rows, heads + 2 * kv, dim), dtype=torch.float16, device=DEV)
        q, k, v = x.split([heads, kv, kv], 1)
        qr, out = torch.empty((rows, heads, dim), dtype=torch.float16, device=DEV), torch.empty((rows, heads, dim), dtype=torch.float16, device=DEV)
        lse = torch.empty((rows, heads), device=DEV)
        a = es.cache_append_t(c, "f16", heads, q.stride()[:2], k.stride()[:2], v.stride()[:2], qr.stride()[:2], freqs.shape[0], dim,
                              "adjacent", prefix)
        d = es.paged_attention_t(c, heads, dim ** -0.5, qr.stride()[:2], out.stride()[:2], True, prefix)
        p = es_program.program_t(km)
        first = p.add_cache_append(a, k_cache, v_cache, k, v, lengths, tables, offsets, dfreqs, q, qr)
        p.add_paged_attention(d, out, qr, k_cache, v_cache, lengths, tables, offsets, lse, shared if prefix else None, deps=[first])
        n = p.finalize()
        ws = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
        p.set_workspace(ws, n)
        return p, x, qr, out, lse, ws

    def verify(x, qr, out, lse, new):
        x, qr, row = x.cpu(), qr.cpu().double(), 0
        for i, n in enumerate(new):
            for r in range(n):
                pos = len(keys[i]) + prefix
                f = freqs[pos].to(torch.complex128)
                keys[i].append(turned(x[row + r, heads:heads + kv].double(), f, dim, False).half().double())
                vals[i].append(x[row + r, heads + kv:].double())
            kk, vv = torch.stack(keys[i]), torch.stack(vals[i])
            if prefix:
                kk, vv = torch.cat([pk.double(), kk]), torch.cat([pv.double(), vv])
            for r in range(n):
                seen = kk.shape[0] - n + r + 1
                for h in range(heads):
                    s = (kk[:seen, h // (heads // kv)] @ qr[row + r, h]) * dim ** -0.5
                    w = torch.softmax(s, 0) @ vv[:seen, h // (heads // kv)]
                    aw = torch.softmax(s, 0) @ vv[:seen, h // (heads // kv)].abs()
                    # half a step of the result, the probabilities' rounding, and one step of each cached key: a
                    # rotation in f32 may round to the f16 beside the exact one's (2^-10 of the key, through q . k)
                    slack = 2 ** -10 * (kk[:seen, h // (heads // kv)].abs() @ qr[row + r, h].abs()).max() * dim ** -0.5
                    tol = 2 ** -11 * w.abs() + (2 ** -11 + 2 * slack) * aw + 2 ** -12
                    assert ((out[row + r, h].cpu().double() - w).abs() <= tol).all()
                    assert abs(lse[row + r, h].cpu().double() - torch.logsumexp(s, 0)) <= slack + 1e-5
            row += n

    offsets = torch.tensor([0, 5, 38, 39], dtype=torch.int32, device=DEV)
    p, x, qr, out, lse, ws = plan(39, offsets)
    x.copy_(torch.randn(x.shape, generator=g).half())
    lengths.copy_(torch.tensor(prompts, dtype=torch.int32))
    p.launch()
    torch.cuda.synchronize()
    verify(x, qr, out, lse, prompts)
    p.close()
    p, x, qr, out, lse, ws = plan(3, None)
    for step in range(steps):
        x.copy_(torch.randn(x.shape, generator=g).half())
        lengths += 1
        if step == 0:
            p.launch()
        else:
            if step == 1:
                p.instantiate()
            p.replay()
        torch.cuda.synchronize()
        verify(x, qr, out, lse, [1, 1, 1])
    assert km.device_status() == 0
    p.close()
