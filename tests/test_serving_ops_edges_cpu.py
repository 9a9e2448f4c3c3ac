"""The CPU definitions of the quantised serving operators at the edges of what their documentation
allows."""

import pytest
import torch

from marin_experiments_b200.ops import api

import serving_ops_oracle as O

BF16 = torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("lens,done,count,status", [([-3, 5], [True, False], 1, 8), ([-64, 5], [True, False], 1, 8),
                                                    ([3, -1], [True, True], 1, 8), ([200, 5], [True, True], 1, 2),
                                                    ([3, 5], [True, True], 9, 8), ([3, 5], [True, True], -1, 8),
                                                    ([100, 100], [True, True], 3, 8), ([-3, 5], [False, True], 1, 0)])
def test_tables_release_refuses(lens, done, count, status):
    """A negative length (short of a page too), a request longer than its table, a bad free count, a
    stack too small: a status, and nothing is changed."""
    state = [ints([[5, 4], [2, 7]]), ints(lens), torch.tensor(done), ints([9, 0, 0, 0, 0, 0]), ints([count])]
    before = [t.clone() for t in state]
    assert int(api.block_tables_release(*state, 64)) == status
    if status:
        assert all(torch.equal(a, b) for a, b in zip(state, before))


def long_request(new):
    """A request longer than its table (64 tokens in two pages of 32), beside an ordinary one."""
    c = O.make_cache([64, 40], hkv=1, hd=64, page=32, seed=2)
    c["tables"] = c["tables"][:, :2].contiguous()
    c["lens"][0] = 65
    q = torch.randn(new + 1, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    return c, q, ints([0, new, new + 1])


@pytest.mark.parametrize("new", [1, 3, 64, 65, 67])
def test_attention_of_a_request_longer_than_its_table(new):
    """All of its rows that see a token are NaN, also those whose tokens the table holds."""
    c, q, starts = long_request(new)
    got = api.kv8_attention(q, c["k"], c["v"], c["ks"], c["vs"], c["tables"], c["lens"], starts=starts)
    blind = max(0, new - 65)
    assert not bool(got[:blind].any()) and bool(torch.isnan(got[blind:new]).all()) and bool(torch.isfinite(got[new]).all())
