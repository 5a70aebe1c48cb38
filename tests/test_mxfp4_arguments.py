"""Outputs and workspaces that the MXFP4 calls refuse in front of a launch; no device
needed: host tensors pass for device tensors, and a call that reaches the library
fails its test.
"""

import pytest
import torch

from spiral_amd import ops
from test_cache_arguments import as_device

N, K, M = 24, 64, 20


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "lib", lambda: pytest.fail("the call reached the library"))


def product(**kw):
    """ops.mxfp4_mul_mat of planar matrices of zeros that say they are on the device."""
    w, x = (as_device(torch.zeros(rows * K // 32 * 17, dtype=torch.uint8)) for rows in (N, M))
    return ops.mxfp4_mul_mat(w, N, K, x, M, **{"workspace": as_device(torch.zeros(64, dtype=torch.uint8)), **kw})


def test_outputs_and_workspace_off_the_device(no_launch):
    """Stores to a host address would fault; a strided workspace is shorter than it says."""
    x = as_device(torch.zeros((2, 64), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="device"):
        ops.mxfp4_quantize(x, out=torch.zeros(200, dtype=torch.uint8))
    out = torch.zeros((M, N))
    with pytest.raises(ValueError, match="device"):
        product(out=out)
    for ws, match in ((torch.zeros(64, dtype=torch.uint8), "device"),
                      (as_device(torch.zeros(128, dtype=torch.uint8))[::2], "contiguous")):
        with pytest.raises(ValueError, match=match):
            product(out=as_device(out), workspace=ws)


def test_output_rows_that_overlap(no_launch):
    """A row stride below n_rows was taken for n_rows, past the tensor's end."""
    for out in (torch.zeros((1, N)).expand(M, N), torch.as_strided(torch.zeros(M * N), (M, N), (N - 1, 1))):
        with pytest.raises(ValueError, match="overlap"):
            product(out=as_device(out))
