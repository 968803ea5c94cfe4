"""Where the paged-cache operators can go wrong without a random input showing it: rounding that adds up, weights far
below the largest, what shared memory held before, arrays that are wrong in part, more than one error in a step."""
import pytest
import torch

import einsummable_b200 as es
from paged_util import batch_t, check, truth
from test_gpu_paged import append_inputs, attend, cache_of, desc_of, km  # noqa: F401 (km: the fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def repeated(b, times):
    """`times` sequences with the pages, lengths and rows of b's one sequence."""
    assert b.batch == 1
    n = b.new[0]
    b.new, b.total, b.batch = b.new * times, b.total * times, times
    b.tables, b.lengths = b.tables.repeat(times, 1), b.lengths.repeat(times)
    b.off = [n * i for i in range(times + 1)]
    b.used = b.rows = n * times
    b.row_offsets = torch.tensor(b.off, dtype=torch.int32) if b.row_offsets is not None else None
    b.q, b.out, b.lse = b.q.repeat(times, 1, 1), b.out.repeat(times, 1, 1), b.lse.repeat(times, 1)
    return b


def set_scores(b, scores, values):
    """Key j of the one sequence (or of the prefix) gets the score scores[j] from every query, and the value values[j]."""
    b.scale = 0.125
    b.q.zero_()
    b.q[..., 0] = 8
    n = len(scores)
    pages = (b.prefix_pages if b.prefix else b.tables[0]).long()
    at = torch.arange(n)
    b.k_cache[pages[at // b.page], at % b.page, :, 0] = scores.to(b.k_cache.dtype).unsqueeze(1)
    b.v_cache[pages[at // b.page], at % b.page] = values.to(b.v_cache.dtype).view(n, 1, 1)


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,prefix", [
    ([1], [2000], 8, 2, 64, 0),                  # single tokens, cut among workers
    ([1], [900], 8, 2, 128, 0),                  # a block a key head
    ([1], [2000], 24, 2, 128, 0),                # 12 query heads a key head
    ([1], [2000], 40, 1, 128, 0),                # 40
    ([40], [1961], 8, 2, 64, 0),                 # rows of a prompt
    ([200], [1801], 8, 2, 128, 0),
    ([1] * 70, [-1] * 70, 8, 2, 128, 4000),      # a batch behind a prefix, read once
])
def test_probabilities_are_not_rounded_to_one_f16(km, new, past, heads, kv_heads, dim, prefix):  # noqa: F811
    """Values of the sign of each probability's rounding to f16: the roundings add up to 2^-13 of the result's
    magnitude where each is taken once, and the result itself is small, so that its own rounding hides nothing.
    Every 16th key has the largest score, which is what all kernels measure the others from."""
    b = batch_t(new, past, heads, kv_heads, dim, 16, prefix=prefix, seed=3)
    n = prefix or b.total[0]
    scores = (-0.3 * torch.rand(n, generator=torch.Generator().manual_seed(5))).half().double()
    scores[::16] = 0
    e = torch.exp(scores)
    set_scores(b, scores, torch.where(e.half().double() > e, 1.0, -1.0))
    want = truth(b, causal=False, precise=True)
    b.to(DEV)
    attend(km, b, causal=False)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    check(b, b.out, b.lse, want)


@pytest.mark.parametrize("new,heads,kv_heads,times", [
    (1, 32, 8, 160),   # single tokens: more (sequence, key head)s than workers, so that one worker has a whole one
    (8, 32, 1, 150),   # 256 rows a key head: more than there are blocks
])
def test_many_keys_far_below_one_that_dominates(km, new, heads, kv_heads, times):  # noqa: F811
    """One key with all of the weight and a value of 0, and 30000 keys 15 to 17 below it (weights of 2^-22 to 2^-25)
    that make up the result."""
    n = 30000
    b = batch_t([new], [n - new], heads, kv_heads, 64, 16, seed=4, offsets=new > 1)
    scores = (-15 - 2 * torch.rand(n, generator=torch.Generator().manual_seed(6))).half().double()
    values = torch.ones(n)
    scores[0], values[0] = 0, 0
    set_scores(b, scores, values)
    out, lse, tol, ltol = truth(b, causal=False, precise=True)
    repeated(b, times).to(DEV)
    attend(km, b, causal=False)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    check(b, b.out, b.lse, tuple(x.repeat(times, *[1] * (x.dim() - 1)) for x in (out, lse, tol, ltol)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [0, 900])
def test_the_same_bits_whatever_ran_before(km, dim, prefix):  # noqa: F811
    """Single tokens with row offsets: 4 of a tile's 8 query rows do not exist.  Calls whose tiles are full, with
    queries that move the maximum all the time or not at all, leave their rows in shared memory."""
    past = [3000, 10, 700, 64, 1999, 830, 1500, 411]
    b = batch_t([1] * 8, past, 8, 2, dim, 16, seed=6, offsets=True, prefix=prefix).to(DEV)
    before = batch_t([2] * 8, past, 8, 2, dim, 16, seed=7, offsets=True, prefix=prefix).to(DEV)
    seen = []
    for factor in (0, 100, 0, 1000, 30):
        keep = before.q.clone()
        before.q *= factor
        attend(km, before)
        before.q = keep
        attend(km, b)
        torch.cuda.synchronize()
        seen.append((b.out.clone(), b.lse.clone()))
    for out, lse in seen[1:]:
        assert torch.equal(out, seen[0][0]) and torch.equal(lse, seen[0][1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 70, 700])
@pytest.mark.parametrize("many", [1, 30])
def test_bad_row_offsets_leave_the_other_sequences_right(km, dtype, prefix, many):  # noqa: F811
    for off, valid in [([0, 2, 5, 99], [0, 1]), ([0, 2, 5, 3], [0, 1]), ([-1, 2, 3, 5], [1, 2]), ([0, 2, 2 ** 20, 5], [0]),
                       ([0, 2, 5, -7], [0, 1]), ([0, 3, 1, 0], [0])]:
        off = [x * many for x in off]
        b = batch_t([2 * many, many, 2 * many], [40, 200, 90], 8, 2, 64, 16, dtype=dtype, seed=9, prefix=prefix)
        b.new = [off[i + 1] - off[i] if i in valid else 0 for i in range(3)]
        b.off = off
        rows = [r for i in valid for r in range(off[i], off[i + 1])]
        want = truth(b)
        b.to(DEV)
        b.row_offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
        attend(km, b)
        torch.cuda.synchronize()
        assert km.device_status() == 0x23
        check(b, b.out[rows], b.lse[rows], tuple(x[rows] for x in want))


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (24, 2), (40, 1)])
@pytest.mark.parametrize("scale", [1.0, 1e26])
def test_scores_of_any_size(km, heads, kv_heads, scale):  # noqa: F811
    """Scores of -2 x 10^11 and of -2 x 10^37, the largest that f16 and the scale allow: the one nearest to 0 has all
    of the weight."""
    b = batch_t([1, 1], [300, 40], heads, kv_heads, 64, 16, seed=8)
    b.scale = scale
    b.q.fill_(60000)
    want = torch.zeros_like(b.out)
    for i in range(2):
        at = torch.arange(b.total[i])
        pages = b.tables[i].long()
        b.k_cache[pages[at // 16], at % 16] = -60000.0
        b.k_cache[pages[27 // 16], 27 % 16] = -59008.0
        want[i] = b.v_cache[pages[27 // 16], 27 % 16].repeat_interleave(heads // kv_heads, 0)
    b.to(DEV)
    attend(km, b)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    assert torch.equal(b.out.cpu(), want)
    top = -64 * 60000.0 * 59008.0 * scale
    assert ((b.lse.cpu().double() / top - 1).abs() <= 2.0 ** -17).all()  # 64 sums, scale, log2 e, ln 2: 2^-24 each


def test_every_error_of_a_step_is_reported(km):  # noqa: F811
    """An append with a bad length and an attention with a bad page: one after the other, whichever came first."""
    assert km.device_status() == 0
    b = batch_t([1, 1], [40, 200], 8, 2, 64, 16, seed=9).to(DEV)
    b.tables[1, 3] = b.n_pages
    attend(km, b)
    x = torch.zeros((2, 2, 64), dtype=torch.float16, device=DEV)
    d = es.cache_append_t(cache_of(b), "f16", 0, k_stride=x.stride()[:2], v_stride=x.stride()[:2])
    lengths = torch.tensor([-3, 0], dtype=torch.int32, device=DEV)
    km.cache_append(d, None, b.k_cache, b.v_cache, x, x, lengths, b.tables)
    torch.cuda.synchronize()
    assert sorted([km.device_status(), km.device_status()]) == [0x21, 0x22]
    assert km.device_status() == 0


def test_null_tensors_are_refused(km):  # noqa: F811
    b = batch_t([1], [40], 4, 2, 64, 16, seed=1).to(DEV)
    n = km.paged_attention_workspace(desc_of(b))
    ws = (torch.empty(n, dtype=torch.uint8, device=DEV), n)
    args = [b.out, b.q, b.k_cache, b.v_cache, b.lengths, b.tables]
    for i in range(6):
        with pytest.raises(es.es_error) as e:
            km.paged_attention(desc_of(b), None, *[None if j == i else a for j, a in enumerate(args)], workspace=ws)
        assert e.value.status == 6
    k = torch.zeros((1, 2, 64), dtype=torch.float16, device=DEV)
    d = es.cache_append_t(cache_of(b), "f16", 0, k_stride=k.stride()[:2], v_stride=k.stride()[:2])
    args = [b.k_cache, b.v_cache, k, k, b.lengths, b.tables]
    for i in range(6):
        with pytest.raises(es.es_error) as e:
            km.cache_append(d, None, *[None if j == i else a for j, a in enumerate(args)])
        assert e.value.status == 6


@pytest.mark.parametrize("rotary", [4, 12, 30])
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_elements_behind_the_rotated_part_are_copied(km, rotary, pairing, dtype):  # noqa: F811
    """Bit for bit, whatever their neighbours are: infinities, NaN and zeros of either sign among them."""
    b = batch_t([3], [9], 4, 2, 64, 16, dtype=dtype, seed=2, filler=0.25)
    q, k, v, freqs = append_inputs(b, dtype, rotary, seed=1, packed=False)
    for x in (q, k):
        x[..., rotary + 1] = float("inf")
        x[..., rotary + 2] = -0.0
        x[..., rotary + 3] = -1.0
        x[0, :, rotary + 5] = float("-inf")
    want_q, want_k = q.clone(), k.clone()
    b.to(DEV)
    q, k, v, freqs = (t.to(DEV) for t in (q, k, v, freqs))
    q_out = torch.zeros_like(q)
    d = es.cache_append_t(cache_of(b), dtype, 4, q.stride()[:2], k.stride()[:2], v.stride()[:2], q_out.stride()[:2],
                          freqs.shape[0], rotary, pairing)
    km.cache_append(d, None, b.k_cache, b.v_cache, k, v, b.lengths, b.tables, b.row_offsets, freqs, q, q_out)
    torch.cuda.synchronize()
    assert km.device_status() == 0
    bits = torch.int16 if dtype == "f16" else torch.int32
    pages = b.tables[0].cpu().long()
    got_k = torch.stack([b.k_cache.cpu()[pages[p // 16], p % 16] for p in range(9, 12)])
    for got, want in ((q_out.cpu(), want_q), (got_k, want_k)):
        assert torch.equal(got[..., rotary:].contiguous().view(bits), want[..., rotary:].contiguous().view(bits))


@pytest.mark.parametrize("many", [1, 30])
def test_append_with_bad_row_offsets_serves_the_other_sequences(km, many):  # noqa: F811
    """Sequences whose rows the offsets name are appended, wherever the wrong entries stand; nothing else is written."""
    for off, valid in [([0, 2, 5, 99], [0, 1]), ([0, 2, 5, 3], [0, 1]), ([-1, 2, 3, 5], [1, 2]), ([0, 2, 2 ** 20, 5], [0]),
                       ([0, 2, 5, -7], [0, 1]), ([0, 3, 1, 0], [0]), ([2, 5, 0, 0], [0])]:
        off = [x * many for x in off]
        b = batch_t([2 * many, many, 2 * many], [40, 200, 90], 4, 2, 64, 16, seed=9, filler=0.25)
        q, k, v, _ = append_inputs(b, "f16", 64, seed=8, packed=False)
        want = b.v_cache.clone()
        for i in valid:
            n = off[i + 1] - off[i]
            for r in range(n):
                p = b.total[i] - n + r
                want[b.tables[i, p // 16].long(), p % 16] = v[off[i] + r]
        b.to(DEV)
        k, v = k.to(DEV), v.to(DEV)
        b.row_offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
        d = es.cache_append_t(cache_of(b), "f16", 0, k_stride=k.stride()[:2], v_stride=v.stride()[:2])
        km.cache_append(d, None, b.k_cache, b.v_cache, k, v, b.lengths, b.tables, b.row_offsets)
        torch.cuda.synchronize()
        assert km.device_status() == 0x23
        assert torch.equal(b.v_cache.cpu(), want)
