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
