"""Which products of MXFP4 weights dequantize them once: both sides of the line, at shapes
where the form that is not taken measured 11 to 40 % slower. No device needed."""

import pytest

from spiral_amd import TYPE_MXFP4


@pytest.mark.parametrize("n,k,m,dense", [(4096, 14336, 768, False), (4096, 14336, 1024, False), (14336, 4096, 512, False),
                                         (14336, 4096, 1024, True), (14336, 4096, 2048, True), (4096, 4096, 1024, False),
                                         (7001, 1024, 2049, True), (2500, 512, 1025, True)])
def test_many_rows(spiral_lib, n, k, m, dense):
    need = spiral_lib.spiral_mul_mat_workspace_bytes(TYPE_MXFP4, n, k, m)
    assert (need == n * k * 2) == dense
