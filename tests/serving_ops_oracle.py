"""fp64 definitions and input builders for the tests of the quantised serving operators."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def e4m3_round(x):
    """fp64 values of magnitude <= 448 to the nearest e4m3 value, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0**-60))).clamp_min(-6) - 3)
    return torch.round(x / step) * step


def scale_exponent(amax: float) -> int:
    """Least e in [-110, 120] with amax <= 448 * 2^e."""
    e = -110
    while e < 120 and amax > 448 * 2.0**e:
        e += 1
    return e


def make_cache(lens, *, hkv, hd, page, seed=0, spare=3, spread=0.0, fill=None):
    """A pool of pages in random order that holds the given lengths. Everything that no request owns
    (spare pages, the tails of last pages) is NaN or ``fill``: it must not be read. Returns a dict of
    CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    width = max(max(need), 1) + 1
    order = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.full((pages, hkv, page, hd), float("nan") if fill is None else fill)
    v = k.clone()
    ks = torch.full((pages, hkv), float("nan"))
    vs = ks.clone()
    at = 0
    for r, n in enumerate(lens):
        for c in range(need[r]):
            p = order[at]
            at += 1
            tables[r, c] = p
            m = min(page, n - c * page)
            for x, s in ((k, ks), (v, vs)):
                y = torch.randn(hkv, m, hd, generator=g) * torch.exp2(spread * torch.randn(hkv, 1, 1, generator=g))
                e = torch.tensor([scale_exponent(float(a)) for a in y.abs().amax((1, 2))])
                x[p, :, :m] = y / torch.exp2(e.float())[:, None, None]
                s[p] = torch.exp2(e.float())
    return {"k": k.to(E4M3), "v": v.to(E4M3), "ks": ks, "vs": vs, "tables": tables,
            "lens": torch.tensor(lens, dtype=torch.int32)}


def attention64(q, c, starts=None, scale=None):
    """(out, sum of weight * |value|) in fp64; rows that see nothing are zero."""
    rows, h, hd = q.shape
    hkv, page = c["k"].shape[1:3]
    scale = hd ** -0.5 if scale is None else scale
    st = list(range(rows + 1)) if starts is None else starts
    o, size = torch.zeros(rows, h, hd, dtype=torch.float64), torch.zeros(rows, h, hd, dtype=torch.float64)
    for r, n in enumerate(c["lens"].tolist()):
        for i in range(st[r], st[r + 1]):
            m = n - (st[r + 1] - 1 - i)
            if m <= 0:
                continue
            pg = c["tables"][r, : -(-m // page)].long()
            k, v = ((x[pg].double() * s[pg].double().abs()[..., None, None]).transpose(1, 2).reshape(-1, hkv, hd)[:m]
                    for x, s in ((c["k"], c["ks"]), (c["v"], c["vs"])))
            for head in range(h):
                kv = head // (h // hkv)
                p = torch.softmax(k[:, kv] @ q[i, head].double() * scale, 0)
                o[i, head] = p @ v[:, kv]
                size[i, head] = p @ v[:, kv].abs()
    return o, size


def attention_bound(o, size):
    """bf16 output: half a step (2^-8 of the value). The f16 weights: 2^-11 each, so 2^-11 of
    sum p |v|; the fp32 scores and exponentials stay below as much again for scores up to 2^7
    (2^-24 * 2^7 * 8 accumulated roundings = 2^-14 of a weight)."""
    return 2.0**-8 * o.abs() + 2.0**-10 * size + 1e-30


def w4_64(x, codes, scales):
    """(x @ w^T, |x| @ |w|^T) in fp64 from integer codes [N, K] and bf16 scales."""
    n, k = codes.shape
    w = (codes.double().view(n, scales.shape[1], -1) * scales.double()[..., None]).view(n, k)
    return x.double() @ w.t(), x.double().abs() @ w.abs().t()


def w4_bound(y, size, k):
    """bf16 output: 2^-8 of the value; K fp32 additions of at most 2^-23 of the sum of magnitudes
    each (the tensor core truncates)."""
    return 2.0**-8 * y.abs() + k * 2.0**-23 * size + 1e-30


def silu64(x):
    return x / (1 + torch.exp(-x))


def close(got, want, bound):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    fine = ~torch.isnan(want)
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float((got - want).abs()[fine].max())}"


def ceil_div(a, b):
    return math.ceil(a / b)
