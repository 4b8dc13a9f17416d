"""Sizes of MXFP4 tensors up to the largest int, without a GPU."""
import ctypes as C

import pytest

import pantheon_b200 as pb
from pantheon_b200 import _lib

P = 1 << 20   # an aligned address that no refused call looks at
TOP = 2 ** 31 - 1


@pytest.mark.parametrize("rows, K", [(TOP, 32), (32, TOP), (TOP - 126, 32), (TOP - 127, 32), (TOP, TOP)])
def test_scale_bytes_of_the_largest_sizes(qglib, rows, K):
    b = C.c_uint64()
    assert qglib.qg_mxfp4_sf_bytes(rows, K, C.byref(b)) == 0
    assert b.value == -(-rows // 128) * -(-K // 128) * 512 == pb.mxfp4_sf_bytes(rows, K)


@pytest.mark.parametrize("M, K", [(TOP, 32), (TOP - 126, 32), (4, TOP - 31), (4, TOP - 479)])
def test_sizes_that_do_not_fit_are_refused_both_ways(qglib, M, K):
    assert K % 32 == 0
    assert qglib.qg_quant_mxfp4(P, 0, K, P, P, M, K, None) == _lib.QG_ERR_ARG
    assert "too large" in _lib.last_error()
    assert qglib.qg_dequant_mxfp4(P, P, P, 0, M, K, None) == _lib.QG_ERR_ARG
    assert "too large" in _lib.last_error()
