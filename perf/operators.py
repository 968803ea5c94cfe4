"""The serving operators over a paged cache, as they are measured: their cases, inputs, plain forms
and 64-bit results.

Three operators that a step of generating tokens makes one after the other:

  append   the new tokens' keys (rotated by their positions) and values go into the cache's pages,
           the queries are rotated on the way
  paged    attention of the new tokens' queries to the cached keys of their own sequence
  prefix   the same for a batch whose sequences all continue one long prompt that lies in the cache
           once

`own` chooses between the plain forms (elementary torch operations) and this package's kernels.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TORCH = {"f16": torch.float16, "f32": torch.float32}
SIZE = {"f16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------- cases
# op        append | paged | prefix
# batch     sequences; heads query heads; kv_heads key / value heads; dim head dim; page tokens a page
# new_lo/hi new tokens of a sequence in this call (1/1: generating, one token each)
# past_lo/hi tokens a sequence has in the cache before them (spread over the logarithm)
# prefix    length of the shared prompt; spare: rows of the tensors behind the last sequence
# spread    which lengths the sequences get
def _case(name, op, batch, heads, kv_heads, dim, page, new, past, dtype="f16", prefix=0, spare=0, halves=False, spread=1):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "dtype": dtype,
            "prefix": prefix, "spare": spare, "halves": halves, "spread": spread}


def listed():
    return [
        # one user's next token: a few microseconds, the launch is what counts
        _case("append_one_token", "append", 1, 32, 8, 128, 16, (1, 1), (700, 700)),
        # one token each of a full batch of the 7B layer's shape (32 heads of 128)
        _case("append_batch", "append", 200, 32, 32, 128, 16, (1, 1), (0, 2000)),
        # prompts of different lengths enter the cache, the tensors padded to a multiple of 64 rows
        _case("append_prompts", "append", 6, 32, 32, 128, 16, (100, 4000), (0, 0), spare=37, spread=3),
        # a float32 model's prompts behind cached ones, heads of 64 rotated by halves
        _case("append_f32", "append", 3, 16, 4, 64, 32, (33, 700), (5, 900), dtype="f32", halves=True),
        # one user's next token after a short prompt, every head with keys of its own
        _case("paged_one_short", "paged", 1, 32, 32, 128, 16, (1, 1), (130, 130)),
        # a full batch of single tokens after texts of very different lengths, an unused place among them
        _case("paged_ragged_batch", "paged", 64, 32, 8, 128, 16, (1, 1), (0, 8191), spread=2),
        # two users with very long contexts: the work has to be split along the keys
        _case("paged_long", "paged", 2, 32, 8, 128, 64, (1, 1), (131000, 131070)),
        # a float32 model generating
        _case("paged_f32", "paged", 12, 16, 4, 64, 16, (1, 1), (1, 2900), dtype="f32", spread=4),
        # the next parts of four prompts attend to what is cached before them and, causally, to themselves
        _case("paged_prompt_parts", "paged", 4, 32, 8, 128, 16, (100, 512), (0, 3500), spare=5, spread=5),
        # three continuations of one short question
        _case("prefix_few", "prefix", 3, 32, 8, 128, 16, (1, 1), (1, 60), prefix=500),
        # a batch of users behind one long system prompt
        _case("prefix_batch", "prefix", 64, 32, 8, 128, 16, (1, 1), (0, 500), prefix=16000),
        # many samples of one question, the 7B layer's shape
        _case("prefix_samples", "prefix", 250, 32, 32, 128, 16, (1, 1), (0, 300), prefix=6001, spread=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "paged", "prefix"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (16, 4), (28, 4), (8, 1), (12, 12)])
    c = _case("", op, 1, heads, kv_heads, rng.choice([64, 80, 112, 128]), rng.choice([8, 16, 32, 48, 64, 128]),
              (1, 1), (0, 0), dtype=rng.choice(["f16", "f16", "f16", "f32"]), spread=rng.randrange(1 << 20),
              halves=rng.random() < 0.5)
    del c["name"]
    if op == "append":
        c["batch"] = _log(rng, 1, 256)
        c["past_hi"] = _log(rng, 1, 2000)
        if rng.random() < 0.5:  # prompts, at most 8000 tokens in all
            c["batch"] = min(c["batch"], 32)
            c["new_hi"] = max(1, _log(rng, 8, 8000) // c["batch"])
            c["new_lo"] = max(1, c["new_hi"] // 30)
            c["spare"] = rng.choice([0, 0, 7])
        return c
    # keys of all sequences padded to the longest: at most 2^18 of 8 heads of 128
    most = (1 << 28) // (c["kv_heads"] * c["dim"])
    if op == "paged":
        c["batch"] = _log(rng, 1, 128)
        if c["dtype"] == "f16" and rng.random() < 0.3:  # parts of prompts
            c["batch"] = _log(rng, 1, 8)
            c["new_hi"] = _log(rng, 2, 512)
            c["new_lo"] = max(1, c["new_hi"] // 20)
            c["past_hi"] = _log(rng, 1, 3500)
            c["spare"] = rng.choice([0, 0, 3])
        else:
            c["past_hi"] = min(_log(rng, 1, 130000), most // c["batch"] - 1)
    else:
        c["batch"] = _log(rng, 2, 256)
        c["prefix"] = min(_log(rng, 16, 16000), (8000 * 8192) // (c["batch"] * c["heads"]))
        c["past_hi"] = min(_log(rng, 1, 1000), most // c["batch"] - 1)
        if c["dtype"] == "f32":  # few rows a key head: float32 is served without the tensor cores
            c["batch"] = min(c["batch"], 8)
    return c


def _lengths(case):
    """(new tokens, cached tokens before them) of every sequence: fixed by the case."""
    rnd = random.Random(case["spread"])

    def some(lo, hi):
        n = [_log(rnd, max(lo, 1), hi) if hi > 0 else 0 for _ in range(case["batch"])]
        n[-1] = hi  # the longest is there
        return n

    new, past = some(case["new_lo"], case["new_hi"]), some(case["past_lo"], case["past_hi"])
    if case["past_lo"] == 0:
        past[0] = 0
    if case["op"] != "append" and case["new_hi"] == 1 and case["past_lo"] == 0 and case["batch"] >= 8:
        past[1] = -1  # an unused place of the batch: no keys at all
    return new, past


# --------------------------------------------------------------------------------------- inputs
def _prepared_call(s):
    """The handle, descriptor and workspace that a program keeps between its steps."""
    import einsummable_b200 as es
    c = s["case"]
    km = es.kernel_manager_t(0)
    cache = es.paged_cache_t(c["dtype"], c["batch"], s["rows"], c["kv_heads"], c["dim"], c["page"], s["n_pages"],
                             s["tables"].shape[1], s["k_cache"].stride()[:3], s["v_cache"].stride()[:3])
    s["km"] = km
    if c["op"] == "append":
        s["desc"] = es.cache_append_t(cache, c["dtype"], c["heads"], q_stride=s["q"].stride()[:2], k_stride=s["k"].stride()[:2],
                                      v_stride=s["v"].stride()[:2], q_out_stride=s["q_out"].stride()[:2],
                                      n_positions=s["freqs"].shape[0], rotary_dim=c["dim"],
                                      pairing="halves" if c["halves"] else "adjacent")
        return
    s["desc"] = es.paged_attention_t(cache, c["heads"], s["scale"], q_stride=s["q"].stride()[:2],
                                     out_stride=s["out"].stride()[:2], causal=True, prefix_len=c["prefix"])
    n = km.paged_attention_workspace(s["desc"])
    s["workspace"] = (torch.empty(max(n, 16), dtype=torch.uint8, device=DEV), n) if n else None


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TORCH[c["dtype"]]
    new, past = _lengths(c)
    total = [n + p for n, p in zip(new, past)]
    used = sum(new)
    rows = used + c["spare"]
    width = max(1, max(-(-t // c["page"]) for t in total))
    n_prefix = -(-c["prefix"] // c["page"])
    need = sum(-(-t // c["page"]) for t in total) + n_prefix
    n_pages = need + 3  # a few are free
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)  # pages come in any order

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    s = {"case": c, "rows": rows, "used": used, "n_pages": n_pages, "scale": 1.0 / math.sqrt(c["dim"])}
    # page tables: a row a sequence, places behind its last page hold page 0
    first = n_prefix
    index = torch.zeros(c["batch"], width, dtype=torch.int64)
    for i, t in enumerate(total):
        n = -(-t // c["page"])
        index[i, :n] = torch.arange(first, first + n)
        first += n
    held = torch.arange(width).unsqueeze(0) < torch.tensor([-(-t // c["page"]) for t in total]).unsqueeze(1)
    s["tables"] = torch.where(held.to(DEV), order[index.to(DEV)], torch.zeros((), dtype=torch.int32, device=DEV)).contiguous()
    s["prefix_pages"] = order[:n_prefix].contiguous()
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    s["row_offsets"] = None if c["new_hi"] == 1 and not c["spare"] else torch.tensor(offsets, dtype=torch.int32, device=DEV)
    s["longest_new"] = max(new)
    s["k_cache"] = normal(n_pages, c["page"], c["kv_heads"], c["dim"])
    s["v_cache"] = normal(n_pages, c["page"], c["kv_heads"], c["dim"])
    s["new"], s["total"] = new, total
    if c["op"] == "append":
        # q, k and v side by side, as one projection leaves them
        qkv = normal(rows, c["heads"] + 2 * c["kv_heads"], c["dim"])
        s["q"], s["k"], s["v"] = qkv.split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
        s["q_out"] = normal(rows, c["heads"], c["dim"])
        angle = torch.arange(max(total) + 1, device=DEV, dtype=torch.float64).unsqueeze(1) * (
            10000.0 ** (-torch.arange(0, c["dim"], 2, device=DEV, dtype=torch.float64) / c["dim"]))
        s["freqs"] = torch.polar(torch.ones_like(angle), angle).to(torch.complex64)
    else:
        s["q"] = normal(rows, c["heads"], c["dim"])
        s["out"] = normal(rows, c["heads"], c["dim"])
        s["lse"] = normal(rows, c["heads"], dtype=torch.float32)
    if own:
        _prepared_call(s)
    return s


# ---------------------------------------------------------------------------------- plain forms
def _rows(s):
    """Of every used row: its sequence, its number inside it, its position in the sequence."""
    if s["row_offsets"] is None:
        seq = torch.arange(s["used"], device=DEV)
        return seq, torch.zeros_like(seq), s["lengths"].long() - 1
    off = s["row_offsets"].long()
    row = torch.arange(s["used"], device=DEV)
    seq = torch.searchsorted(off[1:], row, right=True)
    at = row - off[seq]
    return seq, at, s["lengths"].long()[seq] - (off[seq + 1] - off[seq]) + at


def _rotate(x, f, halves):
    """x [rows, heads, dim] in 32 bits, f [rows, dim / 2] the complex factors of its pairs."""
    re, im = f.real.unsqueeze(1), f.imag.unsqueeze(1)
    if halves:
        a, b = x.chunk(2, -1)
        return torch.cat([a * re - b * im, a * im + b * re], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * re - b * im, a * im + b * re], -1).flatten(-2)


def _plain_append(s):
    c, n = s["case"], s["used"]
    seq, _, pos = _rows(s)
    f = s["freqs"][pos]
    page = s["tables"][seq, pos // c["page"]].long()
    slot = pos % c["page"]
    dt = s["k_cache"].dtype
    s["q_out"][:n] = _rotate(s["q"][:n].float(), f, c["halves"]).to(dt)
    s["k_cache"][page, slot] = _rotate(s["k"][:n].float(), f, c["halves"]).to(dt)
    s["v_cache"][page, slot] = s["v"][:n].to(dt)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _plain_attention(s):
    c, n = s["case"], s["used"]
    b, group, dim, kvh = c["batch"], c["heads"] // c["kv_heads"], c["dim"], c["kv_heads"]
    seq, at, pos = _rows(s)
    wide = s["longest_new"]
    q = torch.zeros(b, wide, kvh, group, dim, device=DEV)
    q[seq, at] = s["q"][:n].float().view(n, kvh, group, dim) * s["scale"]
    see = torch.zeros(b, wide, dtype=torch.int64, device=DEV)  # keys that a row may see
    see[seq, at] = pos + 1
    k = s["k_cache"][s["tables"].long()].flatten(1, 2).float()  # [b, keys, kvh, dim]
    v = s["v_cache"][s["tables"].long()].flatten(1, 2).float()
    keys = k.shape[1]
    x = torch.einsum("bnhgd,bkhd->bhgnk", q, k)
    hidden = torch.arange(keys, device=DEV) >= see.unsqueeze(-1)  # [b, n, keys]
    x = x.masked_fill(hidden[:, None, None], -math.inf)
    if c["prefix"]:
        kp = s["k_cache"][s["prefix_pages"].long()].flatten(0, 1)[:c["prefix"]].float()
        vp = s["v_cache"][s["prefix_pages"].long()].flatten(0, 1)[:c["prefix"]].float()
        x = torch.cat([torch.einsum("bnhgd,khd->bhgnk", q, kp), x], -1)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgnk,bkhd->bnhgd", p[..., c["prefix"]:], v)
    if c["prefix"]:
        o = o + torch.einsum("bhgnk,khd->bnhgd", p[..., :c["prefix"]], vp)
    total, top = total[..., 0].permute(0, 3, 1, 2), top[..., 0].permute(0, 3, 1, 2)  # [b, n, kvh, group]
    o = torch.where(total.unsqueeze(-1) > 0, o / total.unsqueeze(-1), torch.zeros_like(o))
    lse = torch.log(total) + top
    s["out"][:n] = o[seq, at].reshape(n, c["heads"], dim).to(s["out"].dtype)
    s["lse"][:n] = lse[seq, at].reshape(n, c["heads"])
    return s["out"], s["lse"]


def run(s):
    c = s["case"]
    if own:
        stream = torch.cuda.current_stream()
        if c["op"] == "append":
            s["km"].cache_append(s["desc"], stream, s["k_cache"], s["v_cache"], s["k"], s["v"], s["lengths"], s["tables"],
                                 row_offsets=s["row_offsets"], freqs=s["freqs"], q=s["q"], q_out=s["q_out"])
            return s["q_out"], s["k_cache"], s["v_cache"]
        if c["op"] == "paged":
            s["km"].paged_attention(s["desc"], stream, s["out"], s["q"], s["k_cache"], s["v_cache"], s["lengths"], s["tables"],
                                    row_offsets=s["row_offsets"], lse=s["lse"], workspace=s["workspace"])
        else:
            s["km"].prefix_attention(s["desc"], stream, s["out"], s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"],
                                     s["lengths"], s["tables"], row_offsets=s["row_offsets"], lse=s["lse"],
                                     workspace=s["workspace"])
        return s["out"], s["lse"]
    return _plain_append(s) if c["op"] == "append" else _plain_attention(s)


# ------------------------------------------------------------------------------- work and truth
def work(case):
    c, e = case, SIZE[case["dtype"]]
    new, past = _lengths(c)
    used = sum(new)
    if c["op"] == "append":
        moved = 2 * used * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] * e  # q, k, v in; q, k, v out
        angles = sum(new) * c["dim"] // 2 * 8 if c["new_hi"] == 1 else max(n + p for n, p in zip(new, past)) * c["dim"] // 2 * 8
        return {"bytes": moved + angles + 12 * c["batch"], "flops": used * (c["heads"] + c["kv_heads"]) * c["dim"] * 3}
    keys = c["prefix"] + sum(n + p for n, p in zip(new, past))
    pages = -(-keys // c["page"])
    moved = 2 * keys * c["kv_heads"] * c["dim"] * e + 2 * used * c["heads"] * c["dim"] * e + 4 * used * c["heads"]
    seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past)) + used * c["prefix"]
    return {"bytes": moved + 4 * pages + 8 * c["batch"], "flops": 4 * seen * c["heads"] * c["dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    c, half = s["case"], s["case"]["dim"] // 2
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    row = 0
    if c["op"] == "append":
        qo = s["q_out"].double()
        for i, (n, t) in enumerate(zip(s["new"], s["total"])):
            pos = torch.arange(t - n, t, device=DEV)
            f = s["freqs"].to(torch.complex128)[pos].unsqueeze(1)
            page, slot = s["tables"][i].long()[pos // c["page"]], pos % c["page"]

            def turned(x):
                x = x[row:row + n].double()
                z = torch.complex(x[..., :half], x[..., half:]) if c["halves"] else torch.view_as_complex(
                    x.reshape(n, -1, half, 2).contiguous())
                z = z * f
                return torch.cat([z.real, z.imag], -1) if c["halves"] else torch.view_as_real(z).reshape(n, -1, 2 * half)

            qo[row:row + n] = turned(s["q"])
            kc[page, slot] = turned(s["k"])
            vc[page, slot] = s["v"][row:row + n].double()
            row += n
        return qo, kc, vc
    out, lse = s["out"].double(), s["lse"].double()
    group = c["heads"] // c["kv_heads"]
    shared = s["prefix_pages"].long()
    for i, (n, t) in enumerate(zip(s["new"], s["total"])):
        used = s["tables"][i].long()[:-(-t // c["page"])]
        k = torch.cat([kc[shared].flatten(0, 1)[:c["prefix"]], kc[used].flatten(0, 1)[:max(t, 0)]])
        v = torch.cat([vc[shared].flatten(0, 1)[:c["prefix"]], vc[used].flatten(0, 1)[:max(t, 0)]])
        if k.shape[0] == 0:
            out[row:row + n] = 0
            lse[row:row + n] = -math.inf
        else:
            q = s["q"][row:row + n].double().view(n, c["kv_heads"], group, c["dim"]).permute(1, 2, 0, 3).flatten(1, 2)
            x = (q @ k.permute(1, 2, 0) * s["scale"]).view(c["kv_heads"], group, n, -1)
            last = k.shape[0] - n + torch.arange(n, device=DEV)
            x = x.masked_fill(torch.arange(k.shape[0], device=DEV) > last.unsqueeze(1), -math.inf)
            w = torch.softmax(x, -1).flatten(1, 2) @ v.permute(1, 0, 2)
            out[row:row + n] = w.view(c["kv_heads"], group, n, -1).permute(2, 0, 1, 3).reshape(n, c["heads"], -1)
            lse[row:row + n] = torch.logsumexp(x, -1).permute(2, 0, 1).reshape(n, c["heads"])
        row += n
    return out, lse
