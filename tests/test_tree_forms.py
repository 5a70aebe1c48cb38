"""Tree attention with values that are not finite, in every form of its workgroups: one or
two tiles of 16 queries a wave, one to eight query blocks, rows of up to 64, 128 and 256
dims, whole and split over workgroups.
"""

import numpy as np
import pytest
import torch

from test_cache import TYPES, attend, check, make, on, plain

DIMS = [40, 64, 96, 128, 200, 256]
NODES = [5, 12, 25, 40]  # two queries each on a cached head: 1 to 5 tiles


def sees(c, nodes, j):
    """Which of the first tree's nodes see its node j."""
    return (c["mask"][:nodes, 0] >> j & 1).bool().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("nodes", NODES)
@pytest.mark.parametrize("cached", [70, 3000])
def test_rows_that_are_not_finite(cuda, dim, nodes, cached):
    """A drafted row of V, and one of K, with infinities or NaN: no trace in the nodes that
    do not see it; those that do get what the sum gives. Of 3000 cached rows it lies in
    the last of several shares."""
    c = make([cached, 20], [nodes, 8], 4, 2, dim, 16, TYPES[dim // 8 % 2], seed=nodes)
    want, j = plain(c), nodes // 2
    pages, hit, hit_k = c["table"], sees(c, nodes, j), (c["mask"][nodes:, 0] >> 5 & 1).bool().numpy()
    free = np.concatenate([~hit, ~hit_k])
    assert hit.any() and free.any()
    for bad in (float("nan"), float("inf"), -float("inf")):
        d = {n: t.clone() if torch.is_tensor(t) else t for n, t in c.items()}
        d["v"][pages[0, (cached + j) // 16], (cached + j) % 16] = bad
        d["k"][pages[1, 25 // 16], 25 % 16, :, ::3] = bad
        out, lse = attend(on(d, cuda))
        check((out[torch.from_numpy(free)], lse[torch.from_numpy(free)]), [t[free] for t in want])
        got = out[:nodes].double().cpu().numpy()[hit]
        assert np.isnan(got).all() if np.isnan(bad) else (got == bad).all()
        got = lse[:nodes].double().cpu().numpy()
        assert (np.abs(got - want[1][:nodes]) <= want[3][:nodes]).all()  # V has no part in it


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("nodes", NODES)
@pytest.mark.parametrize("cached", [0, 70, 3000])
def test_scores_that_are_nan(cuda, dim, nodes, cached):
    """A NaN in a query makes its own results NaN, one in a cached row those of every node
    of its sequence; zeros and -infinity are for nodes that see no row."""
    c = make([cached, 20], [nodes, 8], 4, 2, dim, 16, TYPES[dim // 8 % 2], seed=nodes)
    want = plain(c)
    d = {n: t.clone() if torch.is_tensor(t) else t for n, t in c.items()}
    d["q"][1, 2, dim // 2] = float("nan")
    d["k"][c["table"][1, 0], 7, 1, 0] = float("nan")  # position 7, the second cached head
    gone = np.zeros(want[1].shape, dtype=bool)
    gone[1, 2] = gone[nodes:, 2:] = True
    out, lse = (t.double().cpu().numpy() for t in attend(on(d, cuda)))
    assert np.isnan(out[gone]).all() and np.isnan(lse[gone]).all()
    assert (np.abs(out - want[0]) <= want[2])[~gone].all() and (np.abs(lse - want[1]) <= want[3])[~gone].all()
