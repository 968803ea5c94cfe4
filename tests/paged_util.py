"""Inputs and a plain 64-bit restatement of the paged-cache operators, shared by their CPU and GPU tests.

Tolerances are bounds, element by element, from the roundings that the operators are allowed:
  * the result is rounded once to its type: half a step, 2^-11 (f16) or 2^-24 (f32) of the value;
  * on the tensor cores the probabilities are rounded to f16 for the product with the values: 2^-11 of
    sum_j p_j |v_j| (the sum of the probabilities is not rounded to f16); with precise=True they are the sum
    of two f16: 2^-22 of sum_j p_j |v_j|, and as their steps are 2^-24 below 2^-14 and the largest of a row is
    at least 2^11, 2^-25 / 2^11 of the row's largest probability for each key: 2^-36 max_j p_j sum_j |v_j|;
  * a score is a sum of d products in f32: off by at most (d + 4) 2^-24 scale sum |q_i k_i|; its factor log2 e and
    the subtraction of the maximum add 2^-22 |s| and the exponential 2^-21; a probability's relative error is
    the sum of these, r, and it enters a normalised result twice: 2 r sum_j p_j |v_j|;
  * sums over n keys in f32 in any order: n 2^-24 of the sum of magnitudes, which for the pairwise and
    per-tile orders here is below (64 + n / 64) 2^-24.
"""
import math

import torch

TORCH = {"f16": torch.float16, "f32": torch.float32}
UNIT = {"f16": 2.0 ** -11, "f32": 2.0 ** -24}


class batch_t:
    """A paged batch: new[i] rows of sequence i behind past[i] cached tokens (past -1: an unused place)."""

    def __init__(self, new, past, heads, kv_heads, dim, page, dtype="f16", prefix=0, spare=0, seed=0, layout="page",
                 offsets=None, device="cpu", filler=float("nan")):
        g = torch.Generator().manual_seed(seed)
        dt = TORCH[dtype]
        self.new, self.total = list(new), [n + p for n, p in zip(new, past)]
        self.heads, self.kv_heads, self.dim, self.page, self.dtype, self.prefix = heads, kv_heads, dim, page, dtype, prefix
        self.batch, self.used = len(new), sum(new)
        self.rows = self.used + spare
        width = max(1, max(-(-t // page) for t in self.total)) + 1  # one more than any sequence needs
        n_prefix = -(-prefix // page)
        self.n_pages = sum(-(-t // page) for t in self.total) + n_prefix + 2
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        # entries behind a sequence's pages are never read: page numbers that do not exist
        self.tables = torch.full((self.batch, width), 1 << 30, dtype=torch.int32)
        first = n_prefix
        for i, t in enumerate(self.total):
            n = -(-t // page)
            self.tables[i, :n] = order[first:first + n]
            first += n
        self.prefix_pages = order[:n_prefix].clone()
        self.lengths = torch.tensor(self.total, dtype=torch.int32)
        off = [0]
        for n in new:
            off.append(off[-1] + n)
        use_offsets = offsets if offsets is not None else (spare > 0 or any(n != 1 for n in new))
        self.row_offsets = torch.tensor(off, dtype=torch.int32) if use_offsets else None
        self.off = off

        def cache():
            if layout == "page":      # [page, slot, head, dim]
                t = torch.randn((self.n_pages, page, kv_heads, dim), generator=g)
            elif layout == "head":    # [page, head, slot, dim]
                t = torch.randn((self.n_pages, kv_heads, page, dim), generator=g).permute(0, 2, 1, 3)
            else:                     # wider than the heads need, an odd number of elements apart
                t = torch.randn((self.n_pages, page, kv_heads, dim + 3), generator=g)[..., :dim]
            return t.to(dt) if layout != "odd" else t.to(dt)

        def pad(t):  # what no token owns holds `filler`
            owned = torch.zeros(self.n_pages, page, dtype=torch.bool)
            for i, n in enumerate(self.total):
                for p in range(max(n, 0)):
                    owned[self.tables[i, p // page].long(), p % page] = True
            for p in range(prefix):
                owned[self.prefix_pages[p // page].long(), p % page] = True
            t[~owned] = filler
            return t

        def strided(t):  # the same values with the layout's strides kept
            if layout == "odd":
                big = torch.zeros((self.n_pages, page, kv_heads, dim + 3), dtype=dt)
                big[..., :dim] = t
                return big[..., :dim]
            return t

        self.k_cache, self.v_cache = strided(pad(cache())), strided(pad(cache()))
        self.q = torch.randn((self.rows, heads, dim), generator=g).to(dt)
        self.out = torch.full((self.rows, heads, dim), 7.0, dtype=dt)
        self.lse = torch.full((self.rows, heads), 7.0, dtype=torch.float32)
        self.scale = 1.0 / math.sqrt(dim)
        self.device = device

    def to(self, device):
        for n in ("tables", "prefix_pages", "lengths", "row_offsets", "q", "out", "lse"):
            t = getattr(self, n)
            setattr(self, n, t.to(device) if t is not None else None)
        for n in ("k_cache", "v_cache"):  # keep the strides
            t = getattr(self, n)
            new = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
            new.copy_(t)
            setattr(self, n, new)
        self.device = device
        return self


def truth(b, causal=True, precise=False):
    """(out, lse, tolerance of out, tolerance of lse), in 64 bits, rows behind the last sequence untouched.
    precise: the probabilities are not allowed a single f16's rounding."""
    kc, vc = b.k_cache.cpu().double(), b.v_cache.cpu().double()
    q = b.q.cpu().double()
    out, lse = b.out.cpu().double(), b.lse.cpu().double()
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    group = b.heads // b.kv_heads
    u, up = UNIT[b.dtype], (UNIT["f16"] if b.dtype == "f16" else 0.0)
    floor = 0.0
    if precise and b.dtype == "f16":
        up, floor = 2.0 ** -22, 2.0 ** -36
    tables, shared = b.tables.cpu().long(), b.prefix_pages.cpu().long()
    for i in range(b.batch):
        for r in range(b.new[i]):
            row = b.off[i] + r
            seen = max(0, b.total[i] - b.new[i] + r + 1) if causal else max(0, b.total[i])
            pos = torch.arange(seen)
            pg, sl = tables[i][pos // b.page], pos % b.page
            pp = torch.arange(b.prefix)
            k = torch.cat([kc[shared[pp // b.page], pp % b.page], kc[pg, sl]])  # [keys, kvh, dim]
            v = torch.cat([vc[shared[pp // b.page], pp % b.page], vc[pg, sl]])
            n = k.shape[0]
            if n == 0:
                out[row], lse[row] = 0, -math.inf
                continue
            qr = q[row].view(b.kv_heads, group, b.dim)
            s = torch.einsum("hgd,khd->hgk", qr, k) * b.scale
            mag = torch.einsum("hgd,khd->hgk", qr.abs(), k.abs()) * abs(b.scale)
            w = torch.softmax(s, -1)
            o = torch.einsum("hgk,khd->hgd", w, v).reshape(b.heads, b.dim)
            av = torch.einsum("hgk,khd->hgd", w, v.abs()).reshape(b.heads, b.dim)
            rel = ((b.dim + 4) * 2.0 ** -24 * mag + 2.0 ** -22 * s.abs()).amax(-1) + 2.0 ** -21  # [kvh, group]
            sums = (64 + n / 64) * 2.0 ** -24
            rel = rel.reshape(b.heads, 1) + sums
            out[row] = o
            tol[row] = u * o.abs() * (1 + 2.0 ** -8) + (up * (1 + 2.0 ** -8) + 2 * rel) * av + (2.0 ** -25 if b.dtype == "f16" else 0)
            if floor:
                least = w.amax(-1, keepdim=True) * v.abs().sum(0).unsqueeze(1)  # [kvh, group, dim]
                tol[row] += floor * least.reshape(b.heads, b.dim)
            lse[row] = torch.logsumexp(s, -1).reshape(b.heads)
            ltol[row] = rel[:, 0] + 2.0 ** -22 * lse[row].abs()
    return out, lse, tol, ltol


def check(b, got_out, got_lse, want):
    out, lse, tol, ltol = want
    err = (got_out.cpu().double() - out).abs()
    bad = ~(err <= tol)
    assert not bad.any(), ("out", int(bad.sum()), err[bad].max().item(), (err / tol.clamp_min(1e-30))[bad].max().item(),
                           bad.nonzero()[:4].tolist())
    if got_lse is not None:
        got = got_lse.cpu().double()
        assert torch.equal(torch.isinf(got), torch.isinf(lse)), "lse of empty rows"
        fin = torch.isfinite(lse)
        bad = ~((got - lse).abs()[fin] <= ltol[fin])
        assert not bad.any(), ("lse", (got - lse).abs()[fin].max().item())
