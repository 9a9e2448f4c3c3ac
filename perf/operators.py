"""Measured cases of the quantised serving path's operators.

Four operators run together in every decode step of a served model: the block tables and slot maps
of the requests (``tables``), the append of new keys and values to a paged cache held in 8 bits
(``append``), attention over that cache (``attention``), and products with 4-bit weights
(``w4``). With ``own`` false each is computed in its plain form (elementary torch operations in
fp32); with ``own`` true by the framework's kernels.

Formats. A cache is ``[pages, kv_heads, page, head_dim]`` of e4m3 with one fp32 power-of-two scale
for each page and head: a value is ``code * scale``. 4-bit weights are int32 words ``[N, K / 8]``:
within each 128 values of a row the 16 words stand in the order 0 4 8 12 1 5 9 13 .. (a 4 x 4
transpose), and a word holds values 0 2 4 6 1 3 5 7 of its eight from the lowest bits up, each as
``code + 8``; a weight is ``code * scale`` with one bf16 scale for each row and ``group`` values.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 128  # rows of one gate (or up) block of a gate/up weight


def listed():
    return [
        # one decode step of a small batch: every request grows by one token
        {"name": "tables-step", "op": "tables", "requests": 8, "page": 64, "context": 4096, "prompts": 0, "rows": 8},
        # a scheduler's step over many requests: most decode, some bring their prompts
        {"name": "tables-mixed", "op": "tables", "requests": 300, "page": 32, "context": 8192, "prompts": 37,
         "rows": 16384},
        # the new token of each request of a small batch
        {"name": "append-step", "op": "append", "requests": 8, "page": 64, "kv_heads": 8, "dim": 128, "most": 1,
         "context": 4096},
        # prompts (and continuations that start inside a page) appended in one call
        {"name": "append-prompts", "op": "append", "requests": 7, "page": 64, "kv_heads": 8, "dim": 128, "most": 2039,
         "context": 300},
        # one user, a short conversation: latency
        {"name": "attn-one", "op": "attention", "requests": 1, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "most": 1, "shortest": 1000, "longest": 1000},
        # a small batch of ragged contexts
        {"name": "attn-batch", "op": "attention", "requests": 8, "page": 64, "heads": 16, "kv_heads": 8, "dim": 128,
         "most": 1, "shortest": 130, "longest": 4096},
        # several tokens a request at once (drafts to verify, the next turn's words), narrow heads
        {"name": "attn-several", "op": "attention", "requests": 24, "page": 32, "heads": 8, "kv_heads": 2, "dim": 64,
         "most": 7, "shortest": 7, "longest": 6001},
        # a full server: many long contexts
        {"name": "attn-long", "op": "attention", "requests": 48, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "most": 1, "shortest": 500, "longest": 32768},
        # the attention output of one token, with the residual
        {"name": "w4-out-1", "op": "w4", "n": 4096, "k": 4096, "group": 128, "tokens": 1, "glu": False,
         "residual": True},
        # gate and up of a batch of eight, with the SwiGLU
        {"name": "w4-gate-up-8", "op": "w4", "n": 24576, "k": 4096, "group": 128, "tokens": 8, "glu": True,
         "residual": False},
        # the down product of a larger, odd batch
        {"name": "w4-down-33", "op": "w4", "n": 4096, "k": 12288, "group": 32, "tokens": 33, "glu": False,
         "residual": True},
        # the output head for four rows
        {"name": "w4-head-4", "op": "w4", "n": 151936, "k": 4096, "group": 64, "tokens": 4, "glu": False,
         "residual": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "w4", "w4"])
    if op == "tables":
        r = _log(rng, 1, 512)
        prompts = rng.randint(0, min(r, 40))
        context = _log(rng, 64, 16384)
        return {"op": op, "requests": r, "page": rng.choice([32, 64, 128]), "context": context, "prompts": prompts,
                "rows": r + prompts * rng.randint(1, 400)}
    if op == "append":
        r = _log(rng, 1, 64)
        return {"op": op, "requests": r, "page": rng.choice([32, 64, 128]), "kv_heads": rng.choice([1, 2, 3, 4, 8]),
                "dim": rng.choice([64, 128]), "most": rng.choice([1, 1, _log(rng, 2, max(3, 14000 // r))]),
                "context": _log(rng, 1, 4096)}
    if op == "attention":
        r, kv = _log(rng, 1, 128), rng.choice([1, 2, 3, 4, 8])
        heads, most = kv * rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 1, rng.randint(2, 8)])
        longest = _log(rng, 1, min(40960, 700_000 // r, 22_000_000 // (r * heads * most)))
        return {"op": op, "requests": r, "page": rng.choice([32, 64, 128]), "heads": heads, "kv_heads": kv,
                "dim": rng.choice([64, 128]), "most": most, "shortest": rng.randint(1, longest), "longest": longest}
    glu = rng.random() < 0.3
    n = 2 * BLOCK * _log(rng, 1, 96) if glu else _log(rng, 17, 40000)
    return {"op": op, "n": n, "k": 128 * _log(rng, 1, 96), "group": rng.choice([32, 64, 128]),
            "tokens": _log(rng, 1, 64), "glu": glu, "residual": not glu and rng.random() < 0.5}


# ------------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, seed):
    """Host lists of the requests' cached and new lengths."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    r = case["requests"]

    def between(lo, hi, n=r):
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()

    if case["op"] == "tables":
        old, new = between(1, case["context"]), [1] * r
        left = case["rows"] - r
        for i in range(case["prompts"]):  # requests that bring a prompt; the first of them are new
            if i % 2 == 0:
                old[i] = 0
            take = min(left, between(0, 2 * left // (case["prompts"] - i), 1)[0])
            new[i] += take
            left -= take
        return old, new
    new = [1 + (i + 1) * (case["most"] - 1) // r for i in range(r)]  # as many in all for every seed
    new = [new[i] for i in torch.randperm(r, generator=g).tolist()]
    if case["op"] == "append":
        return between(0, case["context"]), new
    total = between(case["shortest"], case["longest"])
    total[0] = case["longest"]
    return [max(0, t - n) for t, n in zip(total, new)], new


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def _tables(old, page, width, pool, g):
    """Tables ``[R, width]`` of distinct pages of the pool for the cached lengths (-1 behind them),
    and the free pages in the order of a stack."""
    order = torch.randperm(pool, generator=g, device="cuda").int()
    need = torch.tensor(_pages(old, page), device="cuda")
    first = need.cumsum(0) - need
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp_max(pool - 1)
    tables = torch.where(col < need[:, None], order[at], torch.tensor(-1, dtype=torch.int32, device="cuda"))
    used = int(need.sum())
    free = torch.cat([order[used:], order[:used]])
    return tables.contiguous(), free.contiguous(), pool - used


def _need_exponent(amax):
    """The least e with amax <= 448 * 2^e, in [-110, 120]."""
    m, p = torch.frexp(amax)
    e = torch.where(m <= 0.875, p - 9, p - 8)
    return torch.where(amax > 0, e, torch.full_like(e, -110)).clamp(-110, 120)


def _pool(pages, kv, page, dim, g, outliers):
    """A filled pool: e4m3 codes and their scales. Keys have a few channels that are much larger
    than the others, as after a learned per-head norm."""
    x = torch.randn(pages, kv, page, dim, generator=g, device="cuda")
    if outliers:
        x *= 1 + 6 * (torch.rand(kv, 1, dim, generator=g, device="cuda") > 0.95)
    x *= torch.exp2(torch.randn(pages, kv, 1, 1, generator=g, device="cuda") * 0.5)
    e = _need_exponent(x.abs().amax((2, 3)))
    s = torch.exp2(e.float())
    return (x / s[:, :, None, None]).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    op = case["op"]
    g = _gen(seed)
    if op == "w4":
        n, k, t = case["n"], case["k"], case["tokens"]
        codes = torch.randint(-(2**31), 2**31, (n, k // 8), generator=g, device="cuda").int()
        # no code of -8: weights are rounded to -7 .. 7 steps of their group's largest
        zero = (codes | codes >> 1 | codes >> 2 | codes >> 3) & 0x11111111
        codes = codes | (zero ^ 0x11111111)
        scales = (0.02 / 3 * torch.exp(0.2 * torch.randn(n, k // case["group"], generator=g, device="cuda"))).bfloat16()
        x = torch.randn(t, k, generator=g, device="cuda").bfloat16()
        res = torch.randn(t, n, generator=g, device="cuda").bfloat16() if case["residual"] else None
        return {"op": op, "x": x, "codes": codes, "scales": scales, "residual": res, "glu": case["glu"]}
    old, new = _lengths(case, seed)
    page = case["page"]
    ends = [a + b for a, b in zip(old, new)]
    need = sum(_pages(ends, page))
    if op == "attention":
        width, pool = max(_pages(ends, page)) + 1, need + max(4, need // 8)
    else:  # a server's: any request may grow to its limit
        width = (case["context"] + case.get("rows", case.get("most", 0))) // page + 2
        pool = (case["requests"] * case["context"] + case.get("rows", case.get("most", 0) * case["requests"])) // page
        pool += 2 * case["requests"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if op == "tables":
        tables, free, count = _tables(old, page, width, pool, g)
        return {"op": op, "tables": tables, "lens": ints(old), "new": ints(new), "free": free, "count": ints([count]),
                "page": page, "rows": case["rows"]}
    tables, free, _ = _tables(ends, page, width, pool, g)
    kv, dim = case["kv_heads"], case["dim"]
    k, ks = _pool(pool, kv, page, dim, g, True)
    v, vs = _pool(pool, kv, page, dim, g, False)
    state = {"op": op, "k": k, "v": v, "ks": ks, "vs": vs}
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if op == "append":
        slots = []
        host = tables.tolist()
        for r, (a, b) in enumerate(zip(old, new)):
            slots += [host[r][p // page] * page + p % page for p in range(a, a + b)]
        # as the attention's fused projection gives them: keys contiguous, values a slice of wider rows
        rows = torch.randn(starts[-1], 3 * kv * dim, generator=g, device="cuda").bfloat16()
        state |= {"k_new": rows[:, kv * dim: 2 * kv * dim].reshape(-1, kv, dim).contiguous(),
                  "v_new": rows[:, 2 * kv * dim:].view(-1, kv, dim), "slots": ints(slots)}
        return state
    q = torch.randn(starts[-1], case["heads"], dim, generator=g, device="cuda").bfloat16()
    return state | {"q": q, "tables": tables, "lens": ints(ends), "starts": ints(starts), "most": max(new),
                    "single": case["most"] == 1, "scale": dim ** -0.5}


# -------------------------------------------------------------------------------- plain forms


def _plain_tables(s):
    tables, old, new, free, count, page, rows = (s[k] for k in ("tables", "lens", "new", "free", "count", "page", "rows"))
    dev, r = tables.device, tables.shape[0]
    have, end = (old + page - 1) // page, old + new
    want = (end + page - 1) // page
    more = want - have
    off = more.cumsum(0) - more
    col = torch.arange(tables.shape[1], device=dev)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    at = count - 1 - (off[:, None] + col - have[:, None])
    tables.copy_(torch.where(fresh, free[at.clamp(0, free.shape[0] - 1)], tables))
    starts = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), new.cumsum(0).int()])
    row = torch.arange(rows, device=dev)
    req = torch.searchsorted(starts[1:].contiguous(), row.int(), right=True)
    live = row < starts[-1]
    q = req.clamp_max(r - 1)
    pos = old[q] + row - starts[q]
    slot = tables[q, (pos // page).clamp(0, tables.shape[1] - 1)] * page + pos % page
    minus = torch.full_like(row, -1)
    return {"tables": tables, "lens": end, "free_count": count - more.sum().int(), "starts": starts,
            "slots": torch.where(live, slot, minus).int(), "requests": torch.where(live, req, minus).int(),
            "positions": torch.where(live, pos, torch.zeros_like(row)).int(),
            "status": torch.zeros(1, dtype=torch.int32, device=dev)}


def _plain_store(x, cache, scale, slots):
    pages, kv, page, dim = cache.shape
    live = slots >= 0
    pg, off = (slots // page)[live].long(), (slots % page)[live].long()
    x = x[live].float()
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    amax = torch.zeros(pages, kv, device=x.device).scatter_reduce(0, pg[:, None].expand_as(size), size, "amax")
    first = torch.full((pages,), page, device=x.device).scatter_reduce(0, pg, off, "amin")
    used = first < page
    e = torch.exp2(_need_exponent(amax).float())
    now = torch.where((first == 0)[:, None], e, torch.maximum(e, scale))
    now = torch.where(used[:, None], now, scale)
    tok = torch.arange(page, device=x.device)
    before = (tok < first[:, None]) & used[:, None]
    moved = (cache.float() * (scale / now)[:, :, None, None]).to(cache.dtype)
    new = torch.where(before[:, None, :, None], moved.float(), cache.float()).to(cache.dtype)
    codes = (x / now[pg][:, :, None]).to(cache.dtype)
    new.view(torch.uint8)[pg, :, off] = codes.view(torch.uint8)
    cache.copy_(new)
    scale.copy_(now)


def _plain_append(s):
    _plain_store(s["k_new"], s["k"], s["ks"], s["slots"])
    _plain_store(s["v_new"], s["v"], s["vs"], s["slots"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _plain_attention(s):
    q, tables, lens, starts, most = s["q"], s["tables"], s["lens"], s["starts"], s["most"]
    t, h, dim = q.shape
    kv, page = s["k"].shape[1:3]
    r, width = tables.shape
    pg = tables.clamp_min(0).long()

    def dense(c, sc):  # [R, kv, width * page, dim]
        return (c[pg].float() * sc[pg][..., None, None]).permute(0, 2, 1, 3, 4).reshape(r, kv, width * page, dim)

    i = torch.arange(most, device=q.device)
    count = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp_max(t - 1).long()
    qs = q[row].float().view(r, most, kv, h // kv, dim).permute(0, 2, 1, 3, 4).reshape(r, kv, -1, dim)
    score = qs @ dense(s["k"], s["ks"]).transpose(-1, -2) * s["scale"]
    pos = lens[:, None] - count[:, None] + i
    seen = torch.arange(width * page, device=q.device) <= pos.repeat_interleave(h // kv, 1)[..., None]
    score = score.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    keep = seen.any(1)[:, None, :, None]  # what lies behind a request's end may be anything
    o = p @ torch.where(keep, dense(s["v"], s["vs"]), torch.zeros((), device=q.device))
    o = o.view(r, kv, most, h // kv, dim).permute(0, 2, 1, 3, 4).reshape(r, most, h, dim)
    return o[i < count[:, None]].to(q.dtype)


def _weights(codes, scales):
    n = codes.shape[0]
    w = codes.view(n, -1, 4, 4).transpose(2, 3).reshape(n, -1)  # words in the order of k
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=codes.device)
    v = ((w[..., None] >> shift) & 15).float() - 8
    return (v.view(n, scales.shape[1], -1) * scales.float()[..., None]).view(n, -1)


def _plain_w4(s):
    y = s["x"].float() @ _weights(s["codes"], s["scales"]).t()
    if s["glu"]:
        g = y.view(y.shape[0], -1, 2, BLOCK)
        a, b = g[:, :, 0], g[:, :, 1]
        y = (a / (1 + torch.exp(-a)) * b).reshape(y.shape[0], -1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------------------ the framework


def _own_tables(s):
    from marin_experiments_b200.ops import api

    p = api.block_tables_extend(s["tables"], s["lens"], s["new"], s["free"], s["count"], s["page"], s["rows"])
    return {"tables": s["tables"], "lens": p.lens, "free_count": p.free_count, "starts": p.starts, "slots": p.slots,
            "requests": p.requests, "positions": p.positions, "status": p.status}


def _own_append(s):
    from marin_experiments_b200.ops import api

    api.kv8_append(s["k_new"], s["v_new"], s["k"], s["v"], s["ks"], s["vs"], s["slots"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _own_attention(s):
    from marin_experiments_b200.ops import api

    return api.kv8_attention(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"],
                             starts=None if s["single"] else s["starts"], scale=s["scale"])


def _own_w4(s):
    from marin_experiments_b200.ops import api

    return api.linear_w4(s["x"], s["codes"], s["scales"], residual=s["residual"], glu=s["glu"])


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["op"]](state)


# --------------------------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op == "w4":
        n, k, t = case["n"], case["k"], case["tokens"]
        out = t * (n // 2 if case["glu"] else n)
        return {"bytes": n * k / 2 + 2 * n * k / case["group"] + 2 * t * k + 2 * out + (2 * t * n if case["residual"] else 0),
                "flops": 2.0 * t * n * k}
    old, new = _lengths(case, 1)
    page = case["page"]
    if op == "tables":
        grown = sum(_pages([a + b for a, b in zip(old, new)], page)) - sum(_pages(old, page))
        return {"bytes": 4 * (2 * len(old) + 2 * grown + 2 * len(old) + 3 * case["rows"] + 4), "flops": 0}
    kv, dim = case["kv_heads"], case["dim"]
    if op == "append":  # rows read in 16 bits and written in 8, and the scales of the pages they touch
        touched = sum(-(-(a + b) // page) - a // page for a, b in zip(old, new))
        return {"bytes": 2 * sum(new) * kv * dim * 3 + 4 * sum(new) + 16 * touched * kv, "flops": 4 * sum(new) * kv * dim}
    ends = [a + b for a, b in zip(old, new)]
    h = case["heads"]
    keys = sum(n * e - n * (n - 1) // 2 for n, e in zip(new, ends))
    return {"bytes": 2 * sum(ends) * kv * dim + (8 * kv + 4) * sum(_pages(ends, page)) + 4 * sum(new) * h * dim,
            "flops": 4.0 * keys * h * dim}


# -------------------------------------------------------------------------------------- exact


def _exact_e4m3(x):
    """Round to nearest even of fp64 values of magnitude up to 448 to the e4m3 grid."""
    q = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0**-40))).clamp_min(-6) - 3)
    return torch.round(x / q) * q


def _exact_store(x, cache, scale, slots, page):
    out, sc = cache.double(), scale.double()
    x = x.double()
    at = 0
    while at < len(slots):  # runs of rows in one page
        pg, first = divmod(slots[at], page)
        n = 1
        while at + n < len(slots) and slots[at + n] == slots[at] + n and first + n < page:
            n += 1
        rows = x[at:at + n]
        for h in range(cache.shape[1]):
            e = math.ceil(math.log2(float(rows[:, h].abs().max()) / 448))
            s = 2.0**e if first == 0 else max(2.0**e, float(sc[pg, h]))
            if first:
                out[pg, h, :first] = _exact_e4m3(out[pg, h, :first] * float(sc[pg, h]) / s)
            out[pg, h, first:first + n] = _exact_e4m3(rows[:, h] / s)
            sc[pg, h] = s
        at += n
    return out, sc


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        slots, page = s["slots"].tolist(), case["page"]
        if len(slots) * case["kv_heads"] / min(page, case["most"]) > 3000:
            return None
        k, ks = _exact_store(s["k_new"].cpu(), s["k"].cpu(), s["ks"].cpu(), slots, page)
        v, vs = _exact_store(s["v_new"].cpu(), s["v"].cpu(), s["vs"].cpu(), slots, page)
        return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    if case["op"] == "attention":
        q, lens, starts, tables = s["q"].double(), s["lens"].tolist(), s["starts"].tolist(), s["tables"].long()
        h, dim, kv, page = case["heads"], case["dim"], case["kv_heads"], case["page"]
        out = torch.zeros_like(q)
        for r, n in enumerate(lens):
            pg = tables[r, : -(-n // page)]
            k, v = ((c[pg].double() * sc[pg].double()[..., None, None]).transpose(1, 2).reshape(-1, kv, dim)[:n]
                    for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for j in range(starts[r], starts[r + 1]):
                m = n - (starts[r + 1] - 1 - j)
                qq = q[j].view(kv, h // kv, dim)
                a = torch.softmax(torch.einsum("grd,kgd->grk", qq, k[:m]) / math.sqrt(dim), -1)
                out[j] = torch.einsum("grk,kgd->grd", a, v[:m]).reshape(h, dim)
        return out
    n, k, group = case["n"], case["k"], case["group"]
    x, y = s["x"].double(), []
    for a in range(0, n, 16384):  # value j of a row: 128-block j / 128, word (j % 128) / 8, value j % 8
        c = s["codes"][a:a + 16384].long() & 0xFFFFFFFF
        j = torch.arange(k, device=c.device)
        word = j % 128 // 8
        place = j // 128 * 16 + word % 4 * 4 + word // 4
        nib = (j % 8) // 2 + j % 2 * 4
        w = ((c[:, place] >> (4 * nib)) % 16 - 8).double() * s["scales"][a:a + 16384].double()[:, j // group]
        y.append(x @ w.t())
    y = torch.cat(y, 1)
    if case["glu"]:
        unit = torch.arange(n // 2, device=y.device)
        gate = unit // BLOCK * 2 * BLOCK + unit % BLOCK
        y = torch.nn.functional.silu(y[:, gate]) * y[:, gate + BLOCK]
    return y + s["residual"].double() if case["residual"] else y
