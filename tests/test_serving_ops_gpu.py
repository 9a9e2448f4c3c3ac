"""The quantised serving operators on the GPU (block tables, 8-bit cache append, attention over it,
products with 4-bit weights) against fp64 definitions."""

import pytest
import torch

from marin_experiments_b200.ops import api
from marin_experiments_b200.ops import reference as R
from marin_experiments_b200.ops.quant import unpack_w4

import serving_ops_oracle as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def cuda(c):
    return {k: t.cuda() for k, t in c.items()}


def attend(q, c, **kw):
    return api.kv8_attention(q, c["k"], c["v"], c["ks"], c["vs"], c["tables"], c["lens"], **kw)


# -------------------------------------------------------------------------------- block tables
def tables_state(r, page, seed, longest, grow, slack=5):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, longest + 1, (r,), generator=g).int()
    lens[torch.rand(r, generator=g) < 0.2] = 0
    new = torch.randint(0, grow + 1, (r,), generator=g).int()
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    pool = int(want.sum()) + slack
    order = torch.randperm(pool, generator=g).int()
    tables = torch.full((r, int(want.max()) + 1), -1, dtype=torch.int32)
    at = 0
    for i in range(r):
        n = int(have[i])
        tables[i, :n] = order[at:at + n]
        at += n
    free = torch.full((pool,), -9, dtype=torch.int32)
    free[: pool - at] = order[at:]
    return tables, lens, new, free, torch.tensor([pool - at], dtype=torch.int32)


@pytest.mark.parametrize("r,page,longest,grow,pad", [(1, 64, 0, 1, 0), (1, 32, 63, 1, 3), (8, 64, 300, 1, 0),
                                                     (33, 16, 100, 40, 7), (513, 64, 500, 9, 100),
                                                     (1025, 1, 12, 3, 0), (4096, 128, 700, 2, 5)])
def test_tables_extend(r, page, longest, grow, pad):
    tables, lens, new, free, count = tables_state(r, page, r + page, longest, grow)
    rows = int(new.sum()) + pad
    want_tables = tables.clone()
    want = R.block_tables_extend(want_tables, lens, new, free, count, page, rows)
    args = [t.cuda() for t in (tables, lens, new, free, count)]
    for _ in range(2):  # only the table changes, so a second call gives the same
        got = api.block_tables_extend(*args, page, rows)
        assert int(got.status) == 0
        assert torch.equal(args[0].cpu(), want_tables)
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)
    assert torch.equal(args[1].cpu(), lens) and torch.equal(args[4].cpu(), count)


@pytest.mark.parametrize("case,status", [("pages", 1), ("width", 2), ("rows", 4), ("negative", 8), ("count", 8)])
def test_tables_extend_refuses_on_the_device(case, status):
    tables, lens, new, free, count = tables_state(9, 16, 3, 60, 20, slack=0)
    rows = int(new.sum())
    if case == "pages":
        count -= 1
    elif case == "width":
        tables = tables[:, :-2].contiguous()
    elif case == "rows":
        rows -= 1
    elif case == "negative":
        new[4] = -1
    else:
        count[0] = free.numel() + 1
    want = R.block_tables_extend(tables.clone(), lens, new, free, count, 16, rows)
    args = [t.cuda() for t in (tables, lens, new, free, count)]
    got = api.block_tables_extend(*args, 16, rows)
    assert int(got.status) & status and int(got.status) == int(want[-1])
    assert torch.equal(args[0].cpu(), tables) and torch.equal(got.lens.cpu(), lens)
    assert int(got.free_count) == int(count) and bool((got.slots == -1).all()) and not bool(got.starts.any())


@pytest.mark.parametrize("r,page", [(1, 64), (40, 16), (1000, 32)])
def test_tables_release(r, page):
    tables, lens, _, free, count = tables_state(r, page, 11, 200, 0)
    done = torch.rand(r, generator=torch.Generator().manual_seed(1)) < 0.5
    done[0] = True
    args = [tables.clone(), lens.clone(), done, free.clone(), count.clone()]
    dev = [t.cuda() for t in args]
    assert int(api.block_tables_release(*args, page)) == 0 and int(api.block_tables_release(*dev, page)) == 0
    for a, b in zip(args, dev):
        assert torch.equal(a, b.cpu())
    # a second release of the same requests frees nothing
    assert int(api.block_tables_release(*dev, page)) == 0 and torch.equal(dev[4].cpu(), args[4])


# -------------------------------------------------------------------------------------- append
def same_codes(a, b):
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    assert bool(((a == b) | nan).all())


@pytest.mark.parametrize("hd,hkv,page", [(64, 1, 32), (128, 8, 64), (128, 3, 128), (64, 5, 128)])
@pytest.mark.parametrize("old,new", [([0], [1]), ([0, 31, 32, 5], [1, 1, 1, 1]), ([0, 7, 200, 64], [300, 90, 1, 64]),
                                     ([3] * 40, [1] * 40), ([0], [2500])])
def test_append(hd, hkv, page, old, new):
    ends = [a + b for a, b in zip(old, new)]
    c = O.make_cache(ends, hkv=hkv, hd=hd, page=page, seed=5, fill=0.5)
    c["ks"].nan_to_num_(1.0)
    c["vs"].nan_to_num_(2.0)
    g = torch.Generator().manual_seed(9)
    slots = [int(c["tables"][r, p // page]) * page + p % page for r in range(len(old)) for p in range(old[r], ends[r])]
    slots = torch.tensor(slots + [-1, -1], dtype=torch.int32)
    wide = (torch.randn(slots.numel(), 3 * hkv * hd, generator=g) * torch.exp2(3 * torch.randn(slots.numel(), 1, generator=g))).to(BF16)
    k = wide[:, : hkv * hd].view(-1, hkv, hd)
    v = wide[:, 2 * hkv * hd:].view(-1, hkv, hd)
    d, wd = cuda(c), wide.cuda()
    api.kv8_append(wd[:, : hkv * hd].view(-1, hkv, hd), wd[:, 2 * hkv * hd:].view(-1, hkv, hd), d["k"], d["v"], d["ks"],
                   d["vs"], slots.cuda())
    R.kv8_append(k, v, c["k"], c["v"], c["ks"], c["vs"], slots)
    for n in ("k", "v"):
        same_codes(d[n], c[n])
        assert torch.equal(d[n + "s"].cpu(), c[n + "s"])


def test_append_special_values():
    """Zeros, the largest and smallest bf16 numbers, infinities and NaN."""
    hkv, hd, page = 2, 64, 32
    vals = torch.tensor([0.0, -0.0, 3.3895314e38, 1e-40, float("inf"), -float("inf"), float("nan"), 448.0, 449.0])
    k = torch.zeros(40, hkv, hd)
    for i, x in enumerate(vals):
        k[i, 0, i] = x
        k[32, 1, 0] = x
    k[33:, :, :] = 1e-39
    k, v = k.to(BF16), (k.flip(0) * 0.5).to(BF16)
    c = {"k": torch.zeros(3, hkv, page, hd).to(O.E4M3), "ks": torch.zeros(3, hkv)}
    c |= {"v": c["k"].clone(), "vs": c["ks"].clone()}
    d = cuda(c)
    slots = (torch.arange(40) + 32).int()
    api.kv8_append(k.cuda(), v.cuda(), d["k"], d["v"], d["ks"], d["vs"], slots.cuda())
    R.kv8_append(k, v, c["k"], c["v"], c["ks"], c["vs"], slots)
    for n in ("k", "v"):
        same_codes(d[n], c[n])
        assert torch.equal(d[n + "s"].cpu(), c[n + "s"])


def test_append_token_by_token_is_append_at_once():
    """Scales grow as tokens arrive. Where no code is subnormal the page ends up as from one append."""
    g = torch.Generator().manual_seed(2)
    k = (1 + torch.rand(64, 2, 128, generator=g)) * torch.exp2(torch.arange(64) / 16)[:, None, None]
    k = k.to(BF16).cuda()
    a = {n: torch.zeros(2, 2, 64, 128, device="cuda").to(O.E4M3) for n in "kv"}
    b = {n: torch.zeros(2, 2, 64, 128, device="cuda").to(O.E4M3) for n in "kv"}
    sa = {n: torch.full((2, 2), 7.0, device="cuda") for n in "kv"}
    sb = {n: torch.full((2, 2), 7.0, device="cuda") for n in "kv"}
    slots = torch.arange(64, device="cuda").int() + 64
    api.kv8_append(k, k, a["k"], a["v"], sa["k"], sa["v"], slots)
    for i in range(64):
        api.kv8_append(k[i:i + 1], k[i:i + 1], b["k"], b["v"], sb["k"], sb["v"], slots[i:i + 1])
    assert torch.equal(sa["k"], sb["k"]) and torch.equal(a["k"].view(torch.uint8), b["k"].view(torch.uint8))
    assert float(sa["k"][0, 0]) == 7.0  # the page that no row touches


def test_append_skips_slots_outside_the_cache():
    c = {n: torch.zeros(2, 1, 32, 64, device="cuda").to(O.E4M3) for n in "kv"}
    s = {n: torch.zeros(2, 1, device="cuda") for n in "kv"}
    k = torch.ones(4, 1, 64, device="cuda", dtype=BF16)
    slots = torch.tensor([-1, 64, 2**31 - 1, -(2**31)], dtype=torch.int32, device="cuda")
    api.kv8_append(k, k, c["k"], c["v"], s["k"], s["v"], slots)
    assert not bool(c["k"].float().any()) and not bool(s["v"].any())


# ----------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("hd,h,hkv,page", [(128, 8, 8, 64), (128, 8, 2, 32), (64, 5, 1, 128), (64, 6, 3, 64),
                                           (128, 40, 2, 64), (64, 16, 2, 32)])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2], [31, 32, 33, 127, 128, 129, 0, 255], [700, 5, 1300]])
def test_attention_decode(hd, h, hkv, page, lens):
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=page, seed=len(lens) + h)
    q = torch.randn(len(lens), h, hd, generator=torch.Generator().manual_seed(4)).to(BF16)
    got = attend(q.cuda(), cuda(c))
    want, size = O.attention64(q, c)
    O.close(got, want, O.attention_bound(want, size))


@pytest.mark.parametrize("lens,h,hkv,hd", [([9000], 8, 1, 128), ([4097, 20000], 4, 2, 64), ([50] * 200, 4, 2, 128),
                                           ([1] * 700, 2, 1, 64), ([1500, 129, 40] * 20 + [9000], 4, 2, 128),
                                           ([700] * 130 + [20000], 2, 1, 64)])
def test_attention_splits(lens, h, hkv, hd):
    """Few long requests (many CTAs a segment) and many short ones (many segments a CTA)."""
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=64, seed=1)
    q = torch.randn(len(lens), h, hd, generator=torch.Generator().manual_seed(4)).to(BF16)
    d = cuda(c)
    got = attend(q.cuda(), d)
    want, size = O.attention64(q, c)
    O.close(got, want, O.attention_bound(want, size))
    assert torch.equal(got, attend(q.cuda(), d))  # bit for bit


@pytest.mark.parametrize("h,hkv,hd,page", [(8, 2, 128, 64), (3, 3, 64, 32), (10, 2, 128, 32), (20, 1, 64, 64)])
@pytest.mark.parametrize("lens,new", [([4], [4]), ([40, 0, 33, 500], [3, 0, 33, 1]), ([129, 64, 7], [17, 40, 7]),
                                      ([1, 2, 300], [3, 2, 0])])
def test_attention_several_rows(h, hkv, hd, page, lens, new):
    """Several new rows a request, among them none, all of its tokens, and more than it has tokens."""
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=page, seed=3)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + 5  # padding behind the last request
    wide = torch.randn(rows, 2 * h * hd, generator=torch.Generator().manual_seed(6)).to(BF16)
    q = wide[:, h * hd:].view(rows, h, hd)
    want, size = O.attention64(q, c, starts)
    d, w, st = cuda(c), wide.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda")
    qd = w[:, h * hd:].view(rows, h, hd)
    got = attend(qd, d, starts=st)
    O.close(got, want, O.attention_bound(want, size))
    out = torch.full((rows, h, hd), 7.0, dtype=BF16, device="cuda")
    same = attend(qd, d, starts=st, out=out)
    assert same.data_ptr() == out.data_ptr() and torch.equal(out[: starts[-1]], got[: starts[-1]])
    assert bool((out[starts[-1]:] == 7).all()) and not bool(got[starts[-1]:].any())


def test_attention_scales_far_apart():
    """Pages whose values differ by 2^40, with the weight on the small ones."""
    lens, hkv, hd = [256], 1, 128
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=64, seed=8, spread=20.0)
    q = (0.3 * torch.randn(1, 4, hd, generator=torch.Generator().manual_seed(1))).to(BF16)
    for n, e in enumerate((-30, 10, -20, 0)):
        c["vs"][c["tables"][0, n]] = 2.0**e
        c["ks"][c["tables"][0, n]] = 2.0**(-9 if n != 1 else -3)
    want, size = O.attention64(q, c)
    O.close(attend(q.cuda(), cuda(c)), want, O.attention_bound(want, size))


@pytest.mark.parametrize("factor", [1e-38, 1e-6, 1e6])
def test_attention_query_range(factor):
    """Queries far outside f16's range; the scale brings the scores back."""
    c = O.make_cache([200, 65], hkv=2, hd=64, page=64, seed=9)
    q = (torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)) * factor).to(BF16)
    want, size = O.attention64(q, c, scale=0.1 / factor)
    O.close(attend(q.cuda(), cuda(c), scale=0.1 / factor), want, O.attention_bound(want, size))


def test_attention_bad_pages_and_lengths():
    """A page outside the pool, or a length beyond the table, makes the rows that see it NaN."""
    c = O.make_cache([100, 100, 100, 100, 40], hkv=1, hd=64, page=32, seed=2)
    pages = c["k"].shape[0]
    c["tables"][0, 1], c["tables"][1, 3], c["tables"][2, 0] = pages, -5, 2**31 - 1
    c["lens"][4] = 2**31 - 1
    q = torch.randn(5, 2, 64).to(BF16)
    got = attend(q.cuda(), cuda(c)).cpu()
    ref = R.kv8_attention(q, c["k"], c["v"], c["ks"], c["vs"], c["tables"], c["lens"])
    bad = torch.tensor([True, True, True, False, True])
    assert torch.equal(torch.isnan(got).all(-1).all(-1), bad) and torch.equal(torch.isnan(got), torch.isnan(ref))
    c["lens"][4] = -3
    assert not bool(attend(q.cuda(), cuda(c))[4].any())


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_nan_stays_with_the_rows_that_see_it(hd):
    """A NaN value of token 41, seen by the later of six new rows and by none of the earlier."""
    c = O.make_cache([44, 70], hkv=1, hd=hd, page=32, seed=2)
    v = c["v"].float()
    v[c["tables"][0, 1], 0, 9, 3] = float("nan")
    k = c["k"].float()
    k[c["tables"][1, 2], 0, 4, 5] = float("nan")  # token 68 of the second request: a key
    c["v"], c["k"] = v.to(O.E4M3), k.to(O.E4M3)
    c["vs"][c["tables"][0, 1]] *= -1  # as append marks it
    starts = [0, 6, 10]
    q = torch.randn(10, 3, hd, generator=torch.Generator().manual_seed(1)).to(BF16)
    want, size = O.attention64(q, c, starts)
    assert int(torch.isnan(want).sum()) == 3 * 3 + 2 * 3 * hd  # one column of rows 3..5; rows 8, 9
    got = attend(q.cuda(), cuda(c), starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    O.close(got, want, O.attention_bound(want, size))


@pytest.mark.parametrize("hd,n", [(64, 40), (128, 700)])
def test_attention_of_appended_nan(hd, n):
    """What is not finite in the appended rows reaches exactly the rows that see it, in decode and in
    a call of several rows, in one CTA and in many."""
    hkv, h, page = 2, 4, 64
    pages = -(-n // page)
    c = {"k": torch.zeros(pages, hkv, page, hd).to(O.E4M3), "ks": torch.zeros(pages, hkv)}
    c |= {"v": c["k"].clone(), "vs": c["ks"].clone(), "tables": torch.arange(pages).int()[None].flip(1).contiguous(),
          "lens": torch.tensor([n], dtype=torch.int32)}
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(n, hkv, hd, generator=g), torch.randn(n, hkv, hd, generator=g)
    v[n - 3, 1, 7], v[5, 0, 9], v[5, 0, hd - 1] = float("inf"), float("nan"), float("-inf")
    slots = torch.tensor([int(c["tables"][0, p // page]) * page + p % page for p in range(n)], dtype=torch.int32)
    d = cuda(c)
    api.kv8_append(k.to(BF16).cuda(), v.to(BF16).cuda(), d["k"], d["v"], d["ks"], d["vs"], slots.cuda())
    c = {name: t.cpu() for name, t in d.items()}
    for rows in (1, 5):
        starts = [0, rows]
        q = torch.randn(rows, h, hd, generator=g).to(BF16)
        want, size = O.attention64(q, c, starts)
        assert int(torch.isnan(want).sum()) == rows * 2 * 2 + min(rows, 3) * 2
        got = attend(q.cuda(), d, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
        O.close(got, want, O.attention_bound(want, size))


def test_attention_starts_that_do_not_ascend():
    """Refused on the device: nothing is indexed by them."""
    c = cuda(O.make_cache([40, 50, 60], hkv=1, hd=64, page=32))
    q = torch.randn(8, 2, 64, device="cuda").to(BF16)
    out = torch.full_like(q, 3.0)
    attend(q, c, starts=torch.tensor([0, 8, 2, 8], dtype=torch.int32, device="cuda"), out=out)
    attend(q, c, starts=torch.tensor([-4, 8, 900, 901], dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == 3).all())
    assert not bool(attend(q, c, starts=torch.tensor([0, 8, 2, 8], dtype=torch.int32, device="cuda")).any())
    # rows before the first request belong to none either
    st = torch.tensor([2, 3, 3, 5], dtype=torch.int32, device="cuda")
    got = attend(q, c, starts=st)
    assert not bool(got[:2].any()) and not bool(got[5:].any()) and bool(got[2:5].any(-1).all())


def test_attention_of_a_long_prompt():
    """Hundreds of new rows: many row tiles of one request, each with its own last position."""
    c = O.make_cache([700, 300], hkv=2, hd=64, page=64, seed=5)
    starts = [0, 411, 711]
    q = torch.randn(711, 6, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    want, size = O.attention64(q, c, starts)
    got = attend(q.cuda(), cuda(c), starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    O.close(got, want, O.attention_bound(want, size))


def test_cache_beyond_32_bit_offsets():
    """Append to, and attention over, pages more than 2^32 bytes into the cache."""
    pages, hkv, page, hd = 70_000, 8, 64, 128
    k, v = (torch.empty(pages, hkv, page, hd, dtype=torch.uint8, device="cuda").view(O.E4M3) for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, device="cuda") for _ in range(2))
    table = torch.tensor([[69_999, 3, 66_000]], dtype=torch.int32, device="cuda")
    n = 150
    pos = torch.arange(n, device="cuda")
    slots = (table[0, pos // page] * page + pos % page).int()
    g = torch.Generator().manual_seed(0)
    kn, vn = (torch.randn(n, hkv, hd, generator=g).to(BF16) for _ in range(2))
    api.kv8_append(kn.cuda(), vn.cuda(), k, v, ks, vs, slots)
    small = {"k": torch.zeros(3, hkv, page, hd).to(O.E4M3), "ks": torch.zeros(3, hkv)}
    small |= {"v": small["k"].clone(), "vs": small["ks"].clone(), "tables": torch.tensor([[0, 1, 2]], dtype=torch.int32),
              "lens": torch.tensor([n], dtype=torch.int32)}
    R.kv8_append(kn, vn, small["k"], small["v"], small["ks"], small["vs"], torch.arange(n).int())
    at = table[0].long()
    same_codes(k.view(torch.uint8)[at][2, :, : n - 2 * page], small["k"][2, :, : n - 2 * page])
    assert torch.equal(vs[at].cpu(), small["vs"])
    q = torch.randn(1, 16, hd, generator=g).to(BF16)
    got = api.kv8_attention(q.cuda(), k, v, ks, vs, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    want, size = O.attention64(q, small)
    O.close(got, want, O.attention_bound(want, size))


# -------------------------------------------------------------------------------- 4-bit weights
def w4_case(n, k, group, t, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g)
    scales = (0.02 * torch.exp(0.3 * torch.randn(n, k // group, generator=g))).to(BF16)
    x = torch.randn(t, k, generator=g).to(BF16)
    from marin_experiments_b200.ops.quant import pack_w4

    return codes, pack_w4(codes), scales, x


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,t", [(1, 128, 1), (17, 128, 3), (64, 1152, 8), (100, 2048, 9), (33, 4224, 16),
                                   (16, 256, 31), (250, 384, 33), (40, 1024, 64),
                                     (5000, 256, 5), (70, 12288, 33), (33, 14336, 64), (20, 98304, 3)])
def test_linear_w4(n, k, t, group):
    codes, packed, scales, x = w4_case(n, k, group, t)
    y, size = O.w4_64(x, codes, scales)
    got = api.linear_w4(x.cuda(), packed.cuda(), scales.cuda())
    O.close(got, y, O.w4_bound(y, size, k))
    res = torch.randn(t, n + 3, generator=torch.Generator().manual_seed(1)).to(BF16)
    wide = torch.zeros(t, k + 8, dtype=BF16, device="cuda")
    wide[:, :k] = x.cuda()
    got = api.linear_w4(wide[:, :k], packed.cuda(), scales.cuda(), residual=res.cuda()[:, 3:])
    y = y + res[:, 3:].double()
    O.close(got, y, O.w4_bound(y, size, k) + 2.0**-23 * res[:, 3:].double().abs())


@pytest.mark.parametrize("t", [1, 8, 20, 64])
def test_linear_w4_glu(t):
    codes, packed, scales, x = w4_case(512, 640, 64, t)
    y, size = O.w4_64(x, codes, scales)
    e = 640 * 2.0**-23 * size
    cut = lambda z: (z.view(t, 2, 2, 128)[:, :, 0].reshape(t, -1), z.view(t, 2, 2, 128)[:, :, 1].reshape(t, -1))  # noqa: E731
    (a, b), (ea, eb) = cut(y), cut(e)
    want = O.silu64(a) * b
    # |silu'| < 1.1; fp32's exp and division: 2^-21 of the value
    bound = (2.0**-8 + 2.0**-21) * want.abs() + 1.1 * ea * (b.abs() + eb) + O.silu64(a).abs() * eb + 1e-30
    O.close(api.linear_w4(x.cuda(), packed.cuda(), scales.cuda(), glu=True), want, bound)


@pytest.mark.parametrize("n,glu", [(256, False), (100, False), (512, True)])
def test_linear_w4_many_rows(n, glu):
    """More than 64 rows: bf16 weights on the dense GEMM, each rounded once (2^-8)."""
    t, k = 130, 384
    codes, packed, scales, x = w4_case(n, k, 128, t)
    y, size = O.w4_64(x, codes, scales)
    e = (2.0**-8 + k * 2.0**-23) * size
    if glu:
        cut = lambda z: (z.view(t, -1, 2, 128)[:, :, 0].reshape(t, -1), z.view(t, -1, 2, 128)[:, :, 1].reshape(t, -1))  # noqa: E731
        (a, b), (ea, eb) = cut(y), cut(e)
        y = O.silu64(a) * b
        bound = (2.0**-8 + 2.0**-20) * y.abs() + 1.1 * ea * (b.abs() + eb) + O.silu64(a).abs() * eb
        O.close(api.linear_w4(x.cuda(), packed.cuda(), scales.cuda(), glu=True), y, bound)
        return
    res = torch.randn(t, n, generator=torch.Generator().manual_seed(1)).to(BF16)
    O.close(api.linear_w4(x.cuda(), packed.cuda(), scales.cuda()), y, 2.0**-8 * y.abs() + e)
    # odd widths round the product before the residual is added
    y2 = y + res.double()
    O.close(api.linear_w4(x.cuda(), packed.cuda(), scales.cuda(), residual=res.cuda()), y2,
            2.0**-8 * (y2.abs() + y.abs()) * 1.01 + e * 1.01)


def test_linear_w4_beyond_32_bit_offsets():
    """A matrix of more than 2^32 bytes of codes; its last rows."""
    n, k = 550_000, 16384
    words = torch.randint(-(2**31), 2**31, (1000, k // 8), device="cuda").int()
    codes = torch.empty(n, k // 8, dtype=torch.int32, device="cuda")
    codes[-1000:] = words
    codes[:-1000].zero_()
    scales = torch.full((n, k // 128), 0.01, dtype=BF16, device="cuda")
    x = torch.randn(2, k, device="cuda").to(BF16)
    got = api.linear_w4(x, codes, scales)
    y, size = O.w4_64(x.cpu(), unpack_w4(words.cpu()), scales[-1000:].cpu())
    O.close(got[:, -1000:], y, O.w4_bound(y, size, k))


@pytest.mark.parametrize("t", [8, 40, 70])
def test_linear_w4_of_one_row_repeated(t):
    """An expanded x (row stride 0) gives what its copy gives."""
    _, packed, scales, x = w4_case(200, 1024, 64, 1)
    c, s, x = packed.cuda(), scales.cuda(), x.cuda().expand(t, -1)
    got = api.linear_w4(x, c, s)
    assert torch.equal(got, api.linear_w4(x.contiguous(), c, s))
    assert (got == got[0]).all()


@pytest.mark.parametrize("t", [16, 33, 48, 49, 64])
def test_linear_w4_rows_do_not_mix(t):
    """A NaN in one row of x reaches that row's results alone, and the others keep their bits."""
    _, packed, scales, x = w4_case(300, 2048, 32, t)
    c, s, x = packed.cuda(), scales.cuda(), x.cuda()
    clean = api.linear_w4(x, c, s)
    x[t // 2, 700] = float("nan")
    got = api.linear_w4(x, c, s)
    assert got[t // 2].isnan().all()
    got[t // 2] = clean[t // 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("t", [4, 40])
def test_linear_w4_in_two_graphs_and_streams(t):
    """Graphs with split sums replay beside one another and beside an eager call."""
    _, packed, scales, _ = w4_case(512, 12288, 32, t)
    c, s = packed.cuda(), scales.cuda()
    x = [torch.randn(t, 12288, device="cuda").to(BF16) for _ in range(3)]
    want = [api.linear_w4(v, c, s) for v in x]
    graphs, outs = [], []
    for v in x[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(api.linear_w4(v, c, s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = api.linear_w4(x[2], c, s)
    torch.cuda.synchronize()
    for got, w in zip([*outs, third], want):
        assert torch.equal(got, w)


def test_linear_w4_nan_scale_shows():
    w = torch.randn(32, 256)
    w[5, 130] = float("inf")
    c, s = api.quantize_w4(w.cuda(), 128)
    y = api.linear_w4(torch.randn(2, 256, device="cuda").to(BF16), c, s)
    assert torch.equal(torch.isnan(y).any(0).nonzero().flatten().cpu(), torch.tensor([5]))


def test_quantize_w4_on_the_gpu_is_the_cpu_result():
    w = torch.randn(300, 512).to(BF16)
    for group in (32, 64, 128):
        a, b = api.quantize_w4(w, group), api.quantize_w4(w.cuda(), group, rows=77)
        assert torch.equal(a[0], b[0].cpu()) and torch.equal(a[1], b[1].cpu())


# ------------------------------------------------------------------------------------- together
def test_one_step_together_captured_and_replayed():
    """extend -> append -> attention -> 4-bit product, as a decode step runs them: eagerly, and as a
    captured graph replayed while the lengths grow over page ends."""
    r, h, hkv, hd, page, width, steps = 3, 4, 2, 64, 32, 4, 40
    pool = r * width
    g = torch.Generator().manual_seed(0)
    qs, ks, vs = (torch.randn(steps, r, n, hd, generator=g).to(BF16) for n in (h, hkv, hkv))
    codes, scales = api.quantize_w4(torch.randn(h * hd, h * hd, generator=g) * 0.05, 64)
    cd, sd = codes.cuda(), scales.cuda()

    def state(dev):
        return {"k": torch.zeros(pool, hkv, page, hd, device=dev).to(O.E4M3),
                "v": torch.zeros(pool, hkv, page, hd, device=dev).to(O.E4M3),
                "ks": torch.zeros(pool, hkv, device=dev), "vs": torch.zeros(pool, hkv, device=dev),
                "tables": torch.full((r, width), -1, dtype=torch.int32, device=dev),
                "lens": torch.zeros(r, dtype=torch.int32, device=dev),
                "free": torch.arange(pool, dtype=torch.int32, device=dev),
                "count": torch.tensor([pool], dtype=torch.int32, device=dev),
                "new": torch.ones(r, dtype=torch.int32, device=dev)}

    def step(s, q, k, v, cw, sw):
        p = api.block_tables_extend(s["tables"], s["lens"], s["new"], s["free"], s["count"], page, r)
        s["lens"].copy_(p.lens)
        s["count"].copy_(p.free_count)
        api.kv8_append(k, v, s["k"], s["v"], s["ks"], s["vs"], p.slots)
        o = api.kv8_attention(q, s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"])
        return api.linear_w4(o.view(r, -1), cw, sw, residual=o.view(r, -1))

    eager, graphed, host = state("cuda"), state("cuda"), state("cpu")
    bufs = [qs[0].cuda(), ks[0].cuda(), vs[0].cuda()]
    warm = state("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, *bufs, cd, sd)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed, *bufs, cd, sd)
    for i in range(steps):
        for b, x in zip(bufs, (qs, ks, vs)):
            b.copy_(x[i])
        graph.replay()
        want = step(eager, qs[i].cuda(), ks[i].cuda(), vs[i].cuda(), cd, sd)
        assert torch.equal(out, want), i
        ref = step(host, qs[i], ks[i], vs[i], codes, scales)
        assert float((out.cpu().float() - ref.float()).norm() / ref.float().norm()) < 2.0**-7
    assert torch.equal(graphed["tables"].cpu(), host["tables"]) and int(host["count"]) == pool - 2 * r
    assert torch.equal(graphed["ks"].cpu(), host["ks"])


def test_on_a_side_stream_and_two_calls_at_once():
    """Two streams at the same time, each with its own results (workspaces are per call)."""
    cs = [O.make_cache([3000, 10, 777], hkv=2, hd=128, page=64, seed=s) for s in (1, 2)]
    qs = [torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(s)).to(BF16).cuda() for s in (1, 2)]
    ds = [cuda(c) for c in cs]
    want = [attend(q, d) for q, d in zip(qs, ds)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attend(qs[i], ds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    c = cuda(O.make_cache([40, 50], hkv=2, hd=64, page=32))
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    bad = [lambda: attend(q.float(), c), lambda: attend(q[:, :3], c), lambda: attend(q[:1], c),
           lambda: attend(q, c, starts=torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: attend(q, c, out=q), lambda: attend(q, {**c, "ks": c["ks"][:1]}),
           lambda: attend(q, {**c, "k": c["k"].view(torch.uint8)}), lambda: attend(q, {**c, "lens": c["lens"].long()}),
           lambda: attend(q.transpose(1, 2).contiguous().transpose(1, 2), c),
           lambda: attend(q, {**c, "tables": c["tables"].cpu()}), lambda: attend(q.requires_grad_(), c)]
    k = torch.randn(2, 2, 64, device="cuda").to(BF16)
    slots = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    app = lambda k, v, s: api.kv8_append(k, v, c["k"], c["v"], c["ks"], c["vs"], s)  # noqa: E731
    bad += [lambda: app(k, k[:1], slots), lambda: app(k.float(), k, slots), lambda: app(k, k, slots[:1]),
            lambda: app(k, k, slots.long())]
    codes, scales = api.quantize_w4(torch.randn(256, 256), 64)
    codes, scales = codes.cuda(), scales.cuda()
    x = torch.randn(3, 256, device="cuda").to(BF16)
    bad += [lambda: api.linear_w4(x.float(), codes, scales), lambda: api.linear_w4(x[:, :128], codes, scales),
            lambda: api.linear_w4(x, codes.long(), scales), lambda: api.linear_w4(x, codes, scales[:, :3]),
            lambda: api.linear_w4(x, codes[:128], scales[:128], glu=True),
            lambda: api.linear_w4(x, codes, scales, residual=x[:2]),
            lambda: api.linear_w4(x, codes, scales, residual=x, glu=True),
            lambda: api.linear_w4(x, codes, scales.float())]
    t = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    v = torch.zeros(2, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad += [lambda: api.block_tables_extend(t, v[:1], v, v, one, 32, 4), lambda: api.block_tables_extend(t, v, v, v, v, 32, 4),
            lambda: api.block_tables_extend(t, v, v, v, one, 0, 4), lambda: api.block_tables_extend(t, v, v, v, one, 32, 2**31 - 2),
            lambda: api.block_tables_extend(t, v, v, v, one, 2**30, 4), lambda: api.block_tables_extend(t, v, v, v, one, 32, -1),
            lambda: api.block_tables_release(t, v, v, v, one, 32)]
    for f in bad:
        with pytest.raises((RuntimeError, ValueError)):
            f()
    torch.cuda.synchronize()


def test_empty_calls():
    c = cuda(O.make_cache([40], hkv=2, hd=64, page=32))
    st = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert attend(torch.empty(0, 4, 64, device="cuda", dtype=BF16), c, starts=st).shape == (0, 4, 64)
    k = torch.empty(0, 2, 64, device="cuda", dtype=BF16)
    api.kv8_append(k, k, c["k"], c["v"], c["ks"], c["vs"], st[:0])
    codes, scales = (x.cuda() for x in api.quantize_w4(torch.randn(32, 128), 32))
    assert api.linear_w4(torch.empty(0, 128, device="cuda", dtype=BF16), codes, scales).shape == (0, 32)
