"""Calls of the quantised serving operators at the edges of what their documentation allows, against
fp64 definitions."""

import pytest
import torch

from marin_experiments_b200.ops import api

import serving_ops_oracle as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


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
