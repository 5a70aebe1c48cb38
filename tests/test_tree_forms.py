"""Tree attention with values that are not finite, and with weights far below the largest,
in every form of its workgroups: one or two tiles of 16 queries a wave, one to eight
query blocks, rows of up to 64, 128 and 256 dims, whole and split over workgroups.
"""

import numpy as np
import pytest
import torch

from test_cache import TYPES, U, attend, check, make, on, plain

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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim", [(1, 8), (30, 64), (50, 96), (80, 8), (80, 128), (12, 256), (80, 256)])
@pytest.mark.parametrize("far", [17.3125, 17.34375, 19.0])
def test_many_weights_far_below_the_largest(cuda, far, heads, dim, dtype):
    """One row of score `far` whose value is 0, and 65535 rows of score 0 whose values are 1:
    weights of 2^-25 and 2^-27 of the largest, whose sum is the result. F16 takes them at
    128 times their value, so that each is off by half a step, or by 2^-32 of the
    largest; the rest of the tolerance is that of attention."""
    n, page = 65536, 256
    k, v = torch.zeros((n // page, page, 1, dim), dtype=dtype), torch.ones((n // page, page, 1, dim), dtype=dtype)
    k[0, 0, 0, 0], v[0, 0] = far, 0
    q = torch.zeros((1, heads, dim), dtype=dtype)
    q[:, :, 0] = 1
    c = dict(q=q, k=k, v=v, table=torch.arange(n // page, dtype=torch.int32)[None],
             lens=torch.tensor([n - 1], dtype=torch.int32), cu=torch.tensor([0, 1], dtype=torch.int32),
             mask=torch.tensor([[1]]), max_len=100, max_tree=1)  # too low a length: the rows are not split
    top = float(k[0, 0, 0, 0])
    total = 1 + (n - 1) * np.exp(-top)
    want, lse = (n - 1) * np.exp(-top) / total, top + np.log(total)
    half, d = torch.finfo(dtype).eps / 2, (dim + 4) * U * top + 8 * U
    tol = (2 * d + half + (n + 16) * U) * want + half * want + (2.0 ** -32 * n if dtype == torch.float16 else 0)
    for max_len in (100, n):
        got, z = attend(on({**c, "max_len": max_len}, cuda), scale=1.0)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all(), (got.min(), got.max(), want, tol)
        assert (np.abs(z.double().cpu().numpy() - lse) <= d + n * U + 4 * U * lse).all()
