"""Calls of the quantised serving operators at the edges of what their documentation allows, against
fp64 definitions."""

import os
import subprocess
import sys

import pytest
import torch

from marin_experiments_b200.ops import api

import serving_ops_oracle as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cuda(c):
    return {k: t.cuda() for k, t in c.items()}


def attend(q, c, **kw):
    return api.kv8_attention(q, c["k"], c["v"], c["ks"], c["vs"], c["tables"], c["lens"], **kw)


@pytest.mark.parametrize("h,hkv,hd,lens,new,lead,tail", [
    (32, 8, 128, [4000], [1], 100, 0),                 # one long request, shared by many CTAs
    (32, 8, 128, [4000, 2500], [1, 1], 1, 3),
    (4, 2, 64, [3000, 0, 129, 5000], [3, 0, 2, 9], 17, 5),
    (8, 1, 64, [40, 30], [2, 5], 6, 2),                # short ones, each one CTA's or a cluster's
])
def test_attention_rows_before_the_first_request(h, hkv, hd, lens, new, lead, tail):
    """Rows of no request stay as they were in ``out`` and are zero without it, where several CTAs
    share a request too."""
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=64, seed=11)
    starts = [lead]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + tail
    q = torch.randn(rows, h, hd, generator=torch.Generator().manual_seed(2)).to(BF16)
    want, size = O.attention64(q, c, starts)
    d = cuda(c)
    got = attend(q.cuda(), d, starts=ints(starts))
    O.close(got, want, O.attention_bound(want, size))
    assert not bool(got[:lead].any()) and not bool(got[starts[-1]:].any())
    out = torch.full((rows, h, hd), 7.0, dtype=BF16, device="cuda")
    attend(q.cuda(), d, starts=ints(starts), out=out)
    assert bool((out[:lead] == 7).all()) and bool((out[starts[-1]:] == 7).all())
    assert torch.equal(out[lead:starts[-1]], got[lead:starts[-1]])


def appended(lens, k, v, page):
    """A cache that ``kv8_append`` wrote: request r holds the first ``lens[r]`` of the rows ``k[r]``,
    ``v[r]`` ``[tokens, kv_heads, head_dim]``."""
    hkv, hd = k.shape[2:]
    need = [-(-n // page) for n in lens]
    pages, width = sum(need), max(need)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(7)).int()
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = order[at:at + n]
        at += n
    c = {"k": torch.zeros(pages, hkv, page, hd, device="cuda").to(O.E4M3), "ks": torch.zeros(pages, hkv, device="cuda")}
    c |= {"v": c["k"].clone(), "vs": c["ks"].clone(), "tables": tables.cuda(), "lens": ints(lens)}
    for r, n in enumerate(lens):
        t = torch.arange(n)
        slots = tables[r, t // page] * page + t % page
        api.kv8_append(k[r, :n].to(BF16).cuda(), v[r, :n].to(BF16).cuda(), c["k"], c["v"], c["ks"], c["vs"],
                       slots.int().cuda())
    return c


# (requests, kv heads, tokens): long requests shared among all CTAs, a step of 128 keys each and many steps
# each; clusters of 8 whose CTAs take three steps each; clusters of one CTA.
SPLITS = [(2, 2, 5000), (40, 8, 3000), (4, 8, 3008), (37, 8, 1100)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("r,hkv,n", SPLITS)
@pytest.mark.parametrize("first,zeros,mean,size", [(128, 256, 1.0, 1.0), (512, 512, 0.0, 4.0), (128, 256, 1.0, 1e4),
                                                   (129, 900, 1.0, 1e-3)])
def test_attention_behind_values_that_are_zero(hd, r, hkv, n, first, zeros, mean, size):
    """Ordinary values, then hundreds of tokens whose values are all zero (their pages have the least
    scale there is), then ordinary ones; again and again over the context."""
    g = torch.Generator().manual_seed(3)
    k = 0.3 * torch.randn(r, n, hkv, hd, generator=g)
    v = size * (mean + torch.randn(r, n, hkv, hd, generator=g))
    t = torch.arange(n)
    v[:, t % (first + zeros) >= first] = 0
    d = appended([n] * r, k, v, 64)
    q = torch.randn(r, hkv, hd, generator=g).to(BF16)
    want, s = O.attention64(q, {x: y.cpu() for x, y in d.items()})
    O.close(attend(q.cuda(), d), want, O.attention_bound(want, s))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("r,hkv,n", SPLITS)
@pytest.mark.parametrize("drop", [-20, -35, -45])
def test_attention_over_scales_that_fall_again_and_again(hd, r, hkv, n, drop):
    """Values of 2^0, 2^drop, 2^(2 drop) by turns of 128 tokens."""
    g = torch.Generator().manual_seed(4)
    k = 0.3 * torch.randn(r, n, hkv, hd, generator=g)
    e = drop * (torch.arange(n) // 128 % 3)
    v = (1 + torch.rand(r, n, hkv, hd, generator=g)) * torch.exp2(e.double()).float()[:, None, None]
    d = appended([n] * r, k, v, 64)
    q = torch.randn(r, hkv, hd, generator=g).to(BF16)
    want, s = O.attention64(q, {x: y.cpu() for x, y in d.items()})
    O.close(attend(q.cuda(), d), want, O.attention_bound(want, s))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("drop", [-8, -16, -28])
def test_attention_of_small_values_behind_large_ones(hd, drop):
    """The weight on values far smaller than those before them in the cache, which a fall of the sums'
    unit by 2^56 in all must keep."""
    g = torch.Generator().manual_seed(5)
    n, hkv = 1536, 8
    part = torch.arange(n) // 128 % 3
    v = (1 + torch.rand(1, n, hkv, hd, generator=g)) * torch.exp2((drop * part).float())[:, None, None]
    k = 0.02 * torch.randn(1, n, hkv, hd, generator=g)
    k[..., 0] += torch.where(part == 2, 30.0, -30.0)[:, None]
    q = torch.randn(1, hkv, hd, generator=g)
    q[..., 0] = 40.0
    d = appended([n], k, v, 64)
    want, s = O.attention64(q.to(BF16), {x: y.cpu() for x, y in d.items()})
    assert float(want.abs().max()) < 4 * 2.0 ** (2 * drop)
    # the bound's 1e-30 stays below 2^-8 of the least of these values (2^-56)
    O.close(attend(q.to(BF16).cuda(), d), want, O.attention_bound(want, s))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("r,hkv,n", SPLITS)
def test_attention_of_the_largest_values(hd, r, hkv, n):
    """Values of 2^120 and more: a mean of them is finite, whatever their sum is."""
    g = torch.Generator().manual_seed(6)
    k = 0.3 * torch.randn(r, n, hkv, hd, generator=g)
    v = (1 + 0.9 * torch.rand(r, n, hkv, hd, generator=g)) * 2.0**120
    v[:, ::2, :, ::3] *= -1
    d = appended([n] * r, k, v, 64)
    q = torch.randn(r, hkv, hd, generator=g).to(BF16)
    want, s = O.attention64(q, {x: y.cpu() for x, y in d.items()})
    O.close(attend(q.cuda(), d), want, O.attention_bound(want, s))


@pytest.mark.parametrize("starts", [[0, 8, 20], [-2, 3, 8], [0, 4, 9], [-1, -1, 8], [9, 9, 9], [0, 3, 2**31 - 1],
                                    [-(2**31), 0, 2**31 - 1], [0, -(2**31), 8]])
@pytest.mark.parametrize("lens", [[40, 50], [3000, 5000]])
def test_attention_starts_outside_the_rows(starts, lens):
    """Refused on the device, like those that do not ascend: nothing is computed, and without ``out``
    every row is zero."""
    c = O.make_cache(lens, hkv=1, hd=64, page=32, seed=1)
    q = torch.randn(8, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    d = cuda(c)
    out = torch.full((8, 2, 64), 3.0, dtype=BF16, device="cuda")
    attend(q.cuda(), d, starts=ints(starts), out=out)
    assert bool((out == 3).all())
    # what an earlier tensor held is not what comes out
    junk = torch.full((8, 2, 64), 5.0, dtype=BF16, device="cuda")
    del junk
    assert not bool(attend(q.cuda(), d, starts=ints(starts)).any())
    assert not bool(attend(q, c, starts=torch.tensor(starts, dtype=torch.int32)).any())


@pytest.mark.parametrize("lens,done,count", [([-3, 5], [True, False], 1), ([-64, 5], [True, False], 1),
                                             ([3, -1], [True, True], 1), ([200, 5], [True, True], 1),
                                             ([200, -5], [True, True], 3), ([3, 5], [True, True], 9),
                                             ([3, 5], [True, True], -1), ([100, 100], [True, True], 3),
                                             ([-3, 5], [False, True], 1), ([2**31 - 1] * 2, [True, True], 1)])
def test_tables_release_refuses_like_the_cpu(lens, done, count):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    host = [i32([[5, 4], [2, 7]]), i32(lens), torch.tensor(done), i32([9, 0, 0, 0, 0, 0]), i32([count])]
    dev = [t.cuda() for t in host]
    assert int(api.block_tables_release(*dev, 64)) == int(api.block_tables_release(*host, 64))
    for a, b in zip(host, dev):
        assert torch.equal(a, b.cpu())


@pytest.mark.parametrize("more", [0, 300])  # requests: a cluster each, or shared among all CTAs
@pytest.mark.parametrize("new", [1, 3, 64, 65, 67])
def test_attention_of_a_request_longer_than_its_table(new, more):
    """All of its rows that see a token are NaN, on the CPU too."""
    lens = [64, 40] + [33] * more
    c = O.make_cache(lens, hkv=2, hd=64, page=32, seed=2)
    c["tables"] = c["tables"][:, :2].contiguous()
    c["lens"][0] = 65
    starts = [0, new] + [new + 1 + i for i in range(more + 1)]
    q = torch.randn(new + 1 + more, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    want = attend(q, c, starts=torch.tensor(starts, dtype=torch.int32))
    got = attend(q.cuda(), cuda(c), starts=ints(starts)).cpu()
    blind = max(0, new - 65)
    assert bool(torch.isnan(got[blind:new]).all()) and torch.equal(torch.isnan(got), torch.isnan(want))
    assert not bool(got[:blind].any()) and not bool(want[:blind].any())


def test_attention_out_inside_the_rows_of_q():
    """q may be a slice of wider rows: an out that lies behind its first rows overlaps it all the same,
    one that lies between two rows does not."""
    c = cuda(O.make_cache([40, 50, 7], hkv=2, hd=64, page=32))
    h, hd = 4, 64
    buf = torch.randn(3 * 2 * h * hd + 64, device="cuda").to(BF16)
    q = buf[: 3 * 2 * h * hd].view(3, 2 * h * hd)[:, : h * hd].view(3, h, hd)
    want = attend(q, c)
    for at in (0, 8, h * hd - 8, 3 * h * hd):  # the last: behind q.numel() elements from q's start
        with pytest.raises(RuntimeError, match="overlap"):
            attend(q, c, out=buf[at: at + 3 * h * hd].view(3, h, hd))
    wide = torch.randn(3, 4 * h * hd, device="cuda").to(BF16)
    wide[:, : h * hd] = q.reshape(3, -1)
    out = wide.view(-1)[h * hd: 4 * h * hd].view(3, h, hd)
    assert torch.equal(attend(wide[:, : h * hd].view(3, h, hd), c, out=out), want)
    back = wide.view(-1)[h * hd - 8: 4 * h * hd - 8].view(3, h, hd)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(wide[:, : h * hd].view(3, h, hd), c, out=back)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(want, c, out=want)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(q, c, out=c["k"].view(-1).view(BF16)[: 3 * h * hd].view(3, h, hd))


def test_append_to_one_cache_twice():
    """Keys and values need caches of their own."""
    c = cuda(O.make_cache([40], hkv=1, hd=64, page=32))
    k = torch.ones(1, 1, 64, device="cuda", dtype=BF16)
    for a, b, s, t in (("k", "k", "ks", "vs"), ("k", "v", "ks", "ks")):
        with pytest.raises(RuntimeError, match="overlap"):
            api.kv8_append(k, k, c[a], c[b], c[s], c[t], ints([0]))


def exact_w4(n, k, group, t, seed=0):
    """Small whole numbers times powers of two: every sum of fewer than 2^24 / (4 * 8 * 4) values of K is
    exact in fp32, in any order, so a result is the fp64 one rounded once."""
    from marin_experiments_b200.ops.quant import pack_w4

    assert 4 * 8 * 4 * k < 2**24
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g)
    scales = torch.exp2(torch.randint(0, 3, (n, k // group), generator=g).float()).to(BF16)
    x = torch.randint(-4, 5, (t, k), generator=g).to(BF16)
    w = (codes.double().view(n, -1, group) * scales.double()[..., None]).view(n, k)
    res = (torch.randint(-200, 201, (t, n), generator=g) / 2).to(BF16)
    return x, pack_w4(codes), scales, res, x.double() @ w.t()


@pytest.mark.parametrize("t", [65, 130])
@pytest.mark.parametrize("n", [1, 32, 33, 64, 96, 100, 128, 256, 1000])
def test_linear_w4_many_rows_round_once(t, n):
    """The residual is added before the one rounding, at widths that the dense GEMM does not store too."""
    x, codes, scales, res, y = exact_w4(n, 512, 64, t)
    got = api.linear_w4(x.cuda(), codes.cuda(), scales.cuda(), residual=res.cuda())
    assert torch.equal(got.cpu(), (y + res.double()).to(BF16)) and got.is_contiguous()
    wide = torch.zeros(t, n + 5, dtype=BF16, device="cuda")
    wide[:, 5:] = res.cuda()
    assert torch.equal(api.linear_w4(x.cuda(), codes.cuda(), scales.cuda(), residual=wide[:, 5:]), got)
    assert torch.equal(api.linear_w4(x.cuda(), codes.cuda(), scales.cuda()).cpu(), y.to(BF16))


@pytest.mark.parametrize("n,k,t,group", [(20, 98304, 3, 32), (20, 98304, 3, 128), (5, 98304, 20, 64), (300, 98304, 40, 32),
                                         (70, 12288, 33, 32), (33, 14336, 64, 128), (40, 8192, 1, 64), (4096, 4096, 8, 128),
                                         (5000, 1152, 16, 32), (129, 16384, 31, 128)])
def test_linear_w4_is_exact_on_whole_numbers(n, k, t, group):
    """Bit for bit, so that a slice of K left out or taken twice shows at any K (a bound on the rounding
    errors of 98304 additions is as large as a result there)."""
    x, codes, scales, res, y = exact_w4(n, k, group, t)
    c, s = codes.cuda(), scales.cuda()
    assert torch.equal(api.linear_w4(x.cuda(), c, s).cpu(), y.to(BF16))
    assert torch.equal(api.linear_w4(x.cuda(), c, s, residual=res.cuda()).cpu(), (y + res.double()).to(BF16))


@pytest.mark.parametrize("h,hkv,hd,page,lens,new", [
    # tiles of 16 rows, segments shared among all CTAs
    (96, 8, 128, 64, [300] * 20 + [1, 0, 129] * 7, None), (96, 8, 64, 64, [300] * 30 + [1, 0, 129] * 10, None),
    (16, 1, 64, 32, [300] * 440 + [5000], None),
    (8, 2, 128, 64, [6000, 2500], [3, 4]), (8, 2, 64, 32, [6000, 2500], [3, 4]),
    (4, 2, 128, 64, [9000], [8]), (4, 2, 64, 64, [9000], [8]),
    # in clusters of four and of one
    (12, 4, 128, 128, [4000, 130, 33] * 3, [5, 1, 4] * 3), (20, 2, 128, 64, [900] * 90, None),
    # tiles of 32
    (32, 1, 64, 64, [3000, 700], [2, 1])])
def test_attention_tiles_of_many_rows(h, hkv, hd, page, lens, new):
    """9 and more query rows a kv head, over contexts that several CTAs share, with leading and trailing
    rows of no request where there are several a request."""
    c = O.make_cache(lens, hkv=hkv, hd=hd, page=page, seed=21)
    d = cuda(c)
    starts, rows = None, len(lens)
    if new is not None:
        starts = [5]
        for n in new:
            starts.append(starts[-1] + n)
        rows = starts[-1] + 3
    q = torch.randn(rows, h, hd, generator=torch.Generator().manual_seed(2)).to(BF16)
    want, size = O.attention64(q, c, starts)
    st = None if starts is None else ints(starts)
    got = attend(q.cuda(), d, starts=st)
    O.close(got, want, O.attention_bound(want, size))
    assert torch.equal(got, attend(q.cuda(), d, starts=st))  # bit for bit


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hkv,r,new", [(12, 1, 2, 1), (4, 2, 1, 7), (96, 8, 38, 1), (3, 1, 1, 11)])
def test_attention_tiles_of_many_rows_with_nan_and_zeros(h, hkv, hd, r, new):
    """Tokens whose values are zero for 256 tokens at a time, and values that are not finite: one that all
    rows see, one among the newest tokens that the earlier rows do not."""
    g = torch.Generator().manual_seed(8)
    n = 2500 if r < 10 else 700
    k = 0.3 * torch.randn(r, n, hkv, hd, generator=g)
    v = 1 + torch.randn(r, n, hkv, hd, generator=g)
    v[:, torch.arange(n) % 384 >= 128] = 0
    v[0, 130, 0, 5], v[r - 1, n - 3, hkv - 1, hd - 1] = float("inf"), float("nan")
    d = appended([n] * r, k, v, 64)
    starts = [i * new for i in range(r + 1)]
    q = torch.randn(r * new, h, hd, generator=g).to(BF16)
    want, size = O.attention64(q, {x: y.cpu() for x, y in d.items()}, starts)
    rep = h // hkv
    seen = max(0, min(new, 3))  # rows that see the token n - 3
    assert int(torch.isnan(want).sum()) == rep * (new + seen)
    O.close(attend(q.cuda(), d, starts=ints(starts)), want, O.attention_bound(want, size))


FIRST_CALL = """
import torch
from marin_experiments_b200.ops import api, _ext
codes, scales = (t.cuda() for t in api.quantize_w4(torch.randn(256, 256), 64))
x = torch.randn(40, 256, device="cuda").to(torch.bfloat16)
torch.cuda.synchronize()
{how}
flag = _ext.err_flag(x.device)
flag.fill_(61)  # as a wait that gave up in a kernel before
{again}
try:
    _ext.check_kernel_errors()
    raise SystemExit("the record is lost")
except _ext.KernelTimeoutError:
    pass
_ext.check_kernel_errors()  # cleared
want = api.linear_w4(x[:20].contiguous(), codes, scales)
assert (out[:20].float() - want.float()).abs().max() < 0.05 * want.float().abs().max()
"""


@pytest.mark.parametrize("how,again", [
    ("g = torch.cuda.CUDAGraph()\nwith torch.cuda.graph(g):\n    out = api.linear_w4(x, codes, scales)\n"
     "_ext.check_kernel_errors()", "g.replay()"),
    ("with torch.inference_mode():\n    out = api.linear_w4(x, codes, scales)", "")])
def test_the_error_flag_of_a_first_call_that_is_captured_or_in_inference_mode(how, again):
    """The flag of timed-out waits is no graph's memory (a replay would clear it) and no inference
    tensor (which the check could not clear)."""
    code = FIRST_CALL.format(how=how, again=again)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("starts", [False, True])
def test_the_most_requests_of_a_call(starts):
    """4096 requests, among them empty ones and one that is long."""
    r = 4096
    lens = [(7 * i) % 70 for i in range(r)]
    lens[1234] = 4000
    c = O.make_cache(lens, hkv=1, hd=64, page=32, seed=1)
    new = [i % 3 for i in range(r)] if starts else [1] * r
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    q = torch.randn(first[-1], 2, 64, generator=torch.Generator().manual_seed(2)).to(BF16)
    want, size = O.attention64(q, c, first)
    got = attend(q.cuda(), cuda(c), starts=ints(first) if starts else None)
    O.close(got, want, O.attention_bound(want, size))


def test_a_step_without_new_tokens():
    """Nothing is placed, and nothing but the lengths comes out."""
    tables, lens = ints([[5, 4], [6, -1]]), ints([70, 3])
    p = api.block_tables_extend(tables, lens, ints([0, 0]), ints([9, 0]), ints([1]), 64, 0)
    assert int(p.status) == 0 and p.lens.tolist() == [70, 3] and p.starts.tolist() == [0, 0, 0]
    assert int(p.free_count) == 1 and p.slots.numel() == 0 and tables.tolist() == [[5, 4], [6, -1]]


def test_attention_in_two_graphs_beside_an_eager_call():
    """Graphs of shared segments (with workspaces) and of clusters replay beside one another, over lengths
    that change between the replays."""
    c = [cuda(O.make_cache([n, 40, 700], hkv=2, hd=128, page=64, seed=s)) for n, s in ((5000, 1), (5000, 2), (900, 3))]
    q = [torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(s)).to(BF16).cuda() for s in (1, 2, 3)]
    graphs, outs = [], []
    for i in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(q[i], c[i]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for step in range(8):
        for x in c:
            x["lens"].sub_(step)
        want = [attend(q[i], c[i]) for i in range(3)]
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[3]):
            eager = attend(q[0], c[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*outs, eager], [*want, want[0]])), step


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("r,hkv,n", SPLITS)
@pytest.mark.parametrize("size", [2.0**17, 2.0**22, 2.0**26, 2.0**31])
def test_attention_of_very_large_scores(hd, r, hkv, n, size):
    """Scores far beyond 2^24, whole numbers of which fp32 holds only every other and fewer: the weight is
    on the keys of the largest score alone, eight of them with the same."""
    g = torch.Generator().manual_seed(9)
    k = torch.zeros(r, n, hkv, hd)
    k[..., 0] = size / 2 * torch.rand(r, n, hkv, generator=g)
    best = torch.rand(r, hkv, n, generator=g).topk(8, -1).indices
    for i in range(r):
        for j in range(hkv):
            k[i, best[i, j], j, 0] = size
    v = torch.randn(r, n, hkv, hd, generator=g)
    d = appended([n] * r, k, v, 64)
    q = torch.zeros(r, hkv, hd).to(BF16)
    q[..., 0] = 1
    want, s = O.attention64(q, {x: y.cpu() for x, y in d.items()}, scale=1.0)
    O.close(attend(q.cuda(), d, scale=1.0), want, O.attention_bound(want, s))
