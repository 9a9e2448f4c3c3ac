"""The CPU definitions of the quantised serving operators against independent fp64 ones, and their
refusals."""

import pytest
import torch

from marin_experiments_b200.ops import api
from marin_experiments_b200.ops.quant import pack_w4, unpack_w4

import serving_ops_oracle as O

BF16 = torch.bfloat16


def attend(q, c, **kw):
    return api.kv8_attention(q, c["k"], c["v"], c["ks"], c["vs"], c["tables"], c["lens"], **kw)


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def test_tables_extend_by_hand():
    tables = ints([[5, -1, -1], [-1, -1, -1], [2, 7, -1]])
    p = api.block_tables_extend(tables, ints([3, 0, 8]), ints([2, 4, 1]), ints([9, 8, 6, 4, 0, 0]), ints([4]), 4, 9)
    assert tables.tolist() == [[5, 4, -1], [6, -1, -1], [2, 7, 8]]
    assert p.slots.tolist() == [23, 16, 24, 25, 26, 27, 32, -1, -1]
    assert p.requests.tolist() == [0, 0, 1, 1, 1, 1, 2, -1, -1] and p.positions.tolist() == [3, 4, 0, 1, 2, 3, 8, 0, 0]
    assert p.lens.tolist() == [5, 4, 9] and p.starts.tolist() == [0, 2, 6, 7]
    assert int(p.free_count) == 1 and int(p.status) == 0


@pytest.mark.parametrize("lens,new,count,rows,status", [([3, 8], [2, 1], 1, 9, 1), ([3, 8], [2, 5], 4, 9, 2),
                                                        ([3, 8], [2, 1], 4, 2, 4), ([3, -1], [2, 1], 4, 9, 8),
                                                        ([3, 8], [2, -1], 4, 9, 8), ([3, 8], [2, 1], 5, 9, 8)])
def test_tables_extend_refuses(lens, new, count, rows, status):
    tables = ints([[5, -1, -1], [2, 7, -1]])
    before = tables.clone()
    p = api.block_tables_extend(tables, ints(lens), ints(new), ints([9, 8, 6, 4]), ints([count]), 4, rows)
    assert int(p.status) & status and torch.equal(tables, before)
    assert p.lens.tolist() == lens and int(p.free_count) == count and set(p.slots.tolist()) <= {-1}


def test_tables_release_gives_the_pages_back():
    tables, lens, free, count = ints([[5, 4], [6, -1], [2, 7]]), ints([5, 4, 8]), ints([9, 0, 0, 0, 0, 0]), ints([1])
    assert int(api.block_tables_release(tables, lens, torch.tensor([True, False, True]), free, count, 4)) == 0
    assert free.tolist() == [9, 5, 4, 2, 7, 0] and int(count) == 5
    assert lens.tolist() == [0, 4, 0] and tables.tolist() == [[-1, -1], [6, -1], [-1, -1]]
    assert int(api.block_tables_release(tables, ints([0, 4, 90]), torch.tensor([False, False, True]), free, count, 4)) & 2
    assert int(count) == 5


@pytest.mark.parametrize("first", [0, 3, 31])
def test_append_is_the_definition(first):
    page, hkv, hd, n = 32, 2, 64, 40
    g = torch.Generator().manual_seed(first)
    c = O.make_cache([first + n], hkv=hkv, hd=hd, page=page, seed=1, spread=1.0, fill=0.25)
    c["ks"].nan_to_num_(1.0), c["vs"].nan_to_num_(1.0)
    k0, s0 = c["k"].double(), c["ks"].double()
    k = (4 * torch.randn(n, hkv, hd, generator=g)).to(BF16)
    slots = [int(c["tables"][0, p // page]) * page + p % page for p in range(first, first + n)]
    api.kv8_append(k, k, c["k"], c["v"], c["ks"], c["vs"], ints(slots))
    at = 0
    while at < n:
        pg, off = divmod(slots[at], page)
        m = min(page - off, n - at)
        for h in range(hkv):
            s = 2.0 ** O.scale_exponent(float(k[at:at + m, h].abs().max()))
            if off:
                s = max(s, float(s0[pg, h]))
                assert torch.equal(c["k"][pg, h, :off].double(), O.e4m3_round(k0[pg, h, :off] * float(s0[pg, h]) / s))
            assert float(c["ks"][pg, h]) == s
            assert torch.equal(c["k"][pg, h, off:off + m].double(), O.e4m3_round(k[at:at + m, h].double() / s))
        at += m


def test_append_keeps_what_is_not_finite_visible():
    c = {"k": torch.zeros(1, 1, 32, 64).to(O.E4M3), "ks": torch.zeros(1, 1)}
    v, vs = c["k"].clone(), c["ks"].clone()
    k = torch.ones(3, 1, 64)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = float("inf"), float("-inf"), float("nan")
    api.kv8_append(k.to(BF16), k.to(BF16), c["k"], v, c["ks"], vs, ints([0, 1, 2]))
    got = c["k"].float() * c["ks"]
    assert torch.isnan(got).nonzero().tolist() == [[0, 0, 0, 0], [0, 0, 1, 1], [0, 0, 2, 2]]
    assert float(got[0, 0, 0, 1]) == 1.0
    assert float(c["ks"]) > 0 and float(vs) < 0  # a page of values with NaN is marked
    one = torch.ones(1, 1, 64).to(BF16)
    api.kv8_append(one, one, c["k"], v, c["ks"], vs, ints([5]))
    assert float(vs) < 0
    api.kv8_append(one, one, c["k"], v, c["ks"], vs, ints([0]))  # the page begins anew
    assert float(vs) > 0


@pytest.mark.parametrize("lens,new", [([5, 0, 33], None), ([40, 0, 33, 70], [3, 0, 33, 1]), ([1, 20], [3, 2])])
def test_attention_is_the_definition(lens, new):
    c = O.make_cache(lens, hkv=2, hd=64, page=32, seed=1)
    starts = None
    if new is not None:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
    q = torch.randn(len(lens) if new is None else starts[-1] + 2, 6, 64, generator=torch.Generator().manual_seed(0)).to(BF16)
    want, size = O.attention64(q, c, starts)
    got = attend(q, c, starts=None if starts is None else ints(starts))
    O.close(got, want, O.attention_bound(want, size))


def test_attention_bad_pages_are_nan():
    c = O.make_cache([40, 40, 40], hkv=1, hd=64, page=32, seed=1)
    c["tables"][0, 1] = c["k"].shape[0]
    c["tables"][1, 0] = -2
    c["lens"][2] = 32 * c["tables"].shape[1] + 1
    q = torch.randn(3, 1, 64).to(BF16)
    assert bool(torch.isnan(attend(q, c)).all())


@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_round_trip(group):
    w = torch.randn(50, 384, generator=torch.Generator().manual_seed(0))
    w[3, :group] = 0
    codes, scales = api.quantize_w4(w, group)
    c = unpack_w4(codes)
    assert int(c.max()) <= 7 and int(c.min()) >= -7 and torch.equal(pack_w4(c), codes)
    d = api.dequantize_w4(codes, scales)
    s = scales.float().repeat_interleave(group, 1)
    # half a step, or the part of the largest value that a scale rounded down (2^-8) cannot reach
    assert bool(((d - w).abs() <= s * (0.5 + 7 * 2.0**-8) + 1e-12).all())
    assert not bool(d[3, :group].any())
    again = api.quantize_w4(d, group, out=(torch.empty_like(codes), torch.empty_like(scales)))
    assert torch.equal(again[1][:3], (d[:3].view(3, -1, group).abs().amax(-1) / 7).to(BF16))


def test_w4_layout_by_hand():
    """Value v of a row: word (v / 128) * 16 + (v % 32 / 8) * 4 + v % 128 / 32; even values of the
    eight in the low half of the word, odd in the high half."""
    codes = torch.randint(-8, 8, (2, 256), generator=torch.Generator().manual_seed(3))
    words = pack_w4(codes).tolist()
    for r in range(2):
        for v in range(256):
            word = words[r][v // 128 * 16 + v % 32 // 8 * 4 + v % 128 // 32] & 0xFFFFFFFF
            bit = 4 * (v % 8 // 2) + 16 * (v % 2)
            assert ((word >> bit) & 15) - 8 == int(codes[r, v])


@pytest.mark.parametrize("glu", [False, True])
def test_linear_w4_is_the_definition(glu):
    codes = torch.randint(-8, 8, (256, 256), generator=torch.Generator().manual_seed(3))
    scales = (0.02 * (1 + torch.rand(256, 4))).to(BF16)
    x, res = torch.randn(5, 256).to(BF16), torch.randn(5, 256).to(BF16)
    y, size = O.w4_64(x, codes, scales)
    if glu:
        want = O.silu64(y[:, :128]) * y[:, 128:]
        got = api.linear_w4(x, pack_w4(codes), scales, glu=True)
        e = 256 * 2.0**-23 * size
        O.close(got, want, 2.0**-8 * want.abs() * 1.001 + 1.2 * e[:, :128] * (y[:, 128:].abs() + 1) + e[:, 128:] * (y[:, :128].abs() + 1))
    else:
        got = api.linear_w4(x, pack_w4(codes), scales, residual=res)
        O.close(got, y + res.double(), O.w4_bound(y + res.double(), size, 257))


def test_refusals():
    with pytest.raises(ValueError):
        api.quantize_w4(torch.randn(4, 100), 32)
    with pytest.raises(ValueError):
        api.quantize_w4(torch.randn(4, 128), 48)
    with pytest.raises(ValueError):
        api.quantize_w4(torch.randn(4, 128), 64, out=(torch.empty(4, 16), torch.empty(4, 2)))
    with pytest.raises(ValueError):
        api.quantize_w4(torch.randn(128), 64)
    with pytest.raises(ValueError):
        api.block_tables_extend(ints([[1]]), ints([0]), ints([1]), ints([1]), ints([1]), 0, 1)
    codes, scales = api.quantize_w4(torch.randn(4, 128), 32)
    x = torch.randn(2, 128).requires_grad_()
    with pytest.raises(RuntimeError):
        api.linear_w4(x, codes, scales)
    with torch.no_grad():
        assert api.linear_w4(x, codes, scales).shape == (2, 4)
    c = O.make_cache([4], hkv=1, hd=64, page=32)
    with pytest.raises(RuntimeError):
        attend(torch.randn(1, 1, 64).requires_grad_(), c)


def test_engine_refuses_the_quantised_options_without_a_gpu():
    from marin_experiments_b200.serving.server import tiny_engine

    for kw in ({"kv_cache": "fp8"}, {"weights": "int4"}, {"kv_cache": "int8"}, {"weights": "fp4"}):
        with pytest.raises(ValueError):
            tiny_engine("cpu", **kw)
    assert tiny_engine("cpu", kv_cache="bf16", weights="bf16").ready
