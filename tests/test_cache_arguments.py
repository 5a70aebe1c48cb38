"""Arguments that the cache's and the MXFP4 calls refuse in front of a launch, and the
pool of page ids; no device needed: host tensors pass for device tensors, and a call
that reaches the library fails its test.
"""

import pytest
import torch

from spiral_amd import cache
from test_cache import attend, make


class OnDevice(torch.Tensor):
    """A host tensor that says it is on the device."""

    is_cuda = property(lambda self: True)


def as_device(t):
    return torch.Tensor._make_subclass(OnDevice, t)


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(cache, "lib", lambda: pytest.fail("the call reached the library"))


def inputs():
    c = make([5, 6], [2, 2], 2, 1, 16, 4, torch.bfloat16)
    return {n: as_device(t) if torch.is_tensor(t) else t for n, t in c.items()}


def test_rows_that_overlap(no_launch):
    """One row expanded over all sequences has a stride of 0, which no call can pass on."""
    c = inputs()
    for bad in (as_device(torch.zeros((1, 4), dtype=torch.int32).expand(2, -1)),
                as_device(torch.as_strided(torch.zeros(9, dtype=torch.int32), (2, 4), (3, 1)))):
        with pytest.raises(ValueError, match="table.*overlap"):
            attend({**c, "table": bad})
        with pytest.raises(ValueError, match="table.*overlap"):
            cache.compact(c["k"], c["v"], bad, c["lens"], c["table"], c["lens"])
        with pytest.raises(ValueError, match="keep.*overlap"):
            cache.compact(c["k"], c["v"], c["table"], c["lens"], bad, c["lens"])


def test_outputs_and_workspace_off_the_device(no_launch):
    """Stores to a host address would fault; a strided workspace is shorter than it says."""
    c = inputs()
    host = dict(out=torch.empty(4, 2, 16, dtype=torch.bfloat16), lse=torch.empty(4, 2),
                workspace=torch.empty(1 << 16, dtype=torch.uint8))
    for name, t in host.items():
        with pytest.raises(ValueError, match=f"{name}.*device"):
            attend({**c}, **{n: as_device(o) for n, o in host.items() if n != name}, **{name: t})
    with pytest.raises(ValueError, match="workspace.*contiguous"):
        attend(c, **{**{n: as_device(o) for n, o in host.items()}, "workspace": as_device(host["workspace"])[::2]})


def state(pool):
    return pool.free_pages, list(pool._refs)


@pytest.mark.parametrize("held,gone,rows", [([], [0, 1], 1), ([0], [1], 6), ([1], [0], 5), ([0, 2], [1], 8),
                                            ([0, 1], [2], 10)])
def test_fork_of_released_pages_takes_nothing(held, gone, rows):
    """A page that is no longer in use, whole or the last part of the rows: refused, with
    the references and the free pages as they were."""
    pool = cache.PagePool(6, 4)
    ids = pool.alloc(3)
    pool.release([ids[i] for i in gone])
    before = state(pool)
    with pytest.raises(ValueError, match="not in use"):
        pool.fork(ids, rows)
    assert state(pool) == before
    if 0 in held:
        assert pool.fork(ids, 4) == (ids[:1], [], [])


def test_fork_without_a_free_page_takes_nothing():
    pool = cache.PagePool(2, 4)
    ids = pool.alloc(2)
    before = state(pool)
    with pytest.raises(MemoryError):
        pool.fork(ids, 6)
    assert state(pool) == before


@pytest.mark.parametrize("ids", [[0, 1, 5], [0, -1], [1, 6], [0, 1, 1], [2, 2, 2]])
def test_release_of_too_much_gives_nothing_back(ids):
    """An id without a reference, or one more often than it has: refused as a whole."""
    pool = cache.PagePool(6, 4)
    assert pool.alloc(3) == [0, 1, 2]
    pool.fork([2], 4)  # page 2 twice
    before = state(pool)
    with pytest.raises(ValueError, match="not in use"):
        pool.release(ids)
    assert state(pool) == before
    pool.release(i for i in (2, 0, 2))
    assert pool.free_pages == 5
