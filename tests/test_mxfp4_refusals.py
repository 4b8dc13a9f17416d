"""Refusals of the MXFP4 and gated entry points, and the reference statement of the format, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import pantheon_b200 as pb
from pantheon_b200 import _lib
from tests import mxfp4_reference as R

P = 1 << 20   # an aligned address that no refused call looks at


def _refused(code, word):
    assert code == _lib.QG_ERR_ARG
    assert word in _lib.last_error()


def test_quant_refusals(qglib):
    f = qglib.qg_quant_mxfp4
    _refused(f(None, 0, 64, P, P, 4, 64, None), "null")
    _refused(f(P, 0, 64, None, P, 4, 64, None), "null")
    _refused(f(P, 0, 64, P, P, 0, 64, None), "empty")
    _refused(f(P, 0, 64, P, P, 4, 0, None), "empty")
    _refused(f(P, 0, 63, P, P, 4, 64, None), "stride")
    _refused(f(P, 2, 64, P, P, 4, 64, None), "in_type")
    _refused(f(P, 9, 64, P, P, 4, 64, None), "in_type")
    _refused(f(P + 1, 0, 64, P, P, 4, 64, None), "aligned")
    _refused(f(P, 0, 64, P + 8, P, 4, 64, None), "aligned")
    _refused(f(P, 0, 64, P, P + 4, 4, 64, None), "aligned")


def test_dequant_refusals(qglib):
    f = qglib.qg_dequant_mxfp4
    _refused(f(P, None, P, 0, 4, 64, None), "null")
    _refused(f(P, P, P, 0, 4, 48, None), "multiple of 32")
    _refused(f(P, P, P, 3, 4, 64, None), "out_type")
    _refused(f(P, P, P + 2, 0, 4, 64, None), "aligned")
    _refused(f(P, P, P, 0, -4, 64, None), "empty")


def test_gemm_refusals(qglib):
    f = qglib.qg_gemm_mxfp4
    _refused(f(P, P, P, None, P, 0, 4, 4, 64, None), "null")
    _refused(f(P, P, P, P, None, 0, 4, 4, 64, None), "null")
    _refused(f(P, P, P, P, P, 0, 4, 0, 64, None), "empty")
    _refused(f(P, P, P, P, P, 0, 4, 4, 48, None), "multiple of 32")
    _refused(f(P, P + 8, P, P, P, 0, 4, 4, 64, None), "aligned")
    _refused(f(P, P, P + 1, P, P, 0, 4, 4, 64, None), "aligned")
    _refused(f(P, P, P, P, P + 1, 0, 4, 4, 64, None), "aligned")
    _refused(f(P, P, P, P, P + 2, 1, 4, 4, 64, None), "aligned")
    _refused(f(P, P, P, P, P, 4, 4, 4, 64, None), "out_type")


def test_gated_refusals(qglib):
    f = qglib.qg_gemm_gated_mxfp4
    _refused(f(P, P, P, P, P, None, P, None, 0, 0, 4, 32, 64, None), "null")
    _refused(f(P, P, P, P, P, P, P, None, 0, 2, 4, 32, 64, None), "activation")
    _refused(f(P, P, P, P, P, P, P, None, 4, 0, 4, 32, 64, None), "scale buffer")
    _refused(f(P, P, P, P, P, P, P, P, 4, 0, 4, 40, 64, None), "multiple of 32")
    _refused(f(P, P, P, P, P, P, P + 8, P, 4, 0, 4, 32, 64, None), "aligned")
    _refused(f(P, P, P, P, P + 8, P, P, None, 0, 0, 4, 32, 64, None), "aligned")
    _refused(f(P, P, P, P, P, P, P, None, 3, 0, 4, 32, 64, None), "out_type")


def test_scale_bytes(qglib):
    b = C.c_uint64()
    for rows, K in ((1, 1), (128, 128), (129, 129), (28672, 8192), (5, 4128)):
        assert qglib.qg_mxfp4_sf_bytes(rows, K, C.byref(b)) == 0
        assert b.value == R.up(rows, 128) * R.up(K, 128) // 32 == pb.mxfp4_sf_bytes(rows, K)
    _refused(qglib.qg_mxfp4_sf_bytes(0, 32, C.byref(b)), "bad argument")
    with pytest.raises(ValueError):
        pb.mxfp4_sf_bytes(0, 32)


def test_cpu_tensors_are_refused(qglib):
    q = torch.zeros((4, 32), dtype=torch.uint8)
    sf = torch.zeros((512,), dtype=torch.uint8)
    with pytest.raises(ValueError):
        pb.quant_mxfp4(torch.zeros((4, 64)))
    with pytest.raises(ValueError):
        pb.dequant_mxfp4(q, sf)
    with pytest.raises(ValueError):
        pb.gemm_mxfp4(q, sf, q, sf)
    with pytest.raises(ValueError):
        pb.gemm_gated_mxfp4(q, sf, q, sf, q, sf)


def test_reference_rounds_to_the_nearest_level_with_ties_to_even():
    x = np.zeros((1, 32))
    x[0, :12] = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.0, -5.1, 0.26, 0.24]
    code, byte = R.quantise(x)
    assert byte[0, 0] == 127
    assert list(code[0, :12]) == [7, 0, 2, 2, 4, 4, 6, 6, 8, 15, 1, 0]
    q, sf = R.pack(code, byte)
    assert list(R.decode(q, sf)[0, :4]) == [6.0, 0.0, 1.0, 1.0]


@pytest.mark.parametrize("name", ["qg_gemm_gated_bf16", "qg_gemm_gated_f16"])
def test_gated_dense_refusals(qglib, name):
    f = getattr(qglib, name)
    _refused(f(P, P, None, P, None, None, 0, 4, 8, 8, None), "null")
    _refused(f(P, P, P, None, None, None, 0, 4, 8, 8, None), "null")
    _refused(f(P, P, P, P, P, None, 0, 4, 8, 8, None), "together")
    _refused(f(P, P, P, P, None, None, 2, 4, 8, 8, None), "activation")
    _refused(f(P, P, P, P, None, None, 0, 0, 8, 8, None), "empty")
    _refused(f(P, P, P, P, None, None, 0, 4, 12, 8, None), "multiples of 8")
    _refused(f(P, P, P, P, None, None, 0, 4, 8, 12, None), "multiples of 8")
    _refused(f(P, P + 8, P, P, None, None, 0, 4, 8, 8, None), "aligned")
    _refused(f(P, P, P, P + 2, None, None, 0, 4, 8, 8, None), "aligned")
    _refused(f(P, P, P, P, None, None, 0, 1 << 30, 8, 8, None), "too large")


@pytest.mark.parametrize("name", ["qg_gemm_gated_bf16_backward", "qg_gemm_gated_f16_backward"])
def test_gated_backward_refusals(qglib, name):
    f = getattr(qglib, name)
    big = 1 << 30
    _refused(f(None, P, P, P, P, P, P, P, P, 0, 4, 8, 8, P, big, None), "null")
    _refused(f(P, P, P, P, P, None, P, P, P, 0, 4, 8, 8, P, big, None), "null")
    _refused(f(P, P, P, P, P, P, P, P, None, 0, 4, 8, 8, P, big, None), "together")
    _refused(f(P, P, P, P, P, P, None, None, None, 0, 4, 8, 8, P, big, None), "no gradient")
    _refused(f(P, P, P, P, P, P, P, P, P, -1, 4, 8, 8, P, big, None), "activation")
    _refused(f(P, P, P, P, P, P, P, P, P, 0, 4, 8, 20, P, big, None), "multiples of 8")
    _refused(f(P, P, P, P, P, P, P, P, P, 0, 4, 8, 8, None, big, None), "workspace")
    b = C.c_uint64()
    assert qglib.qg_gemm_gated_backward_workspace_bytes(4, 8, C.byref(b)) == 0 and b.value >= 4 * 4 * 8
    _refused(f(P, P, P, P, P, P, P, P, P, 0, 4, 8, 8, P, b.value - 1, None), "workspace")
    _refused(f(P, P, P, P, P, P, P, P, P, 0, 4, 8, 8, P + 8, big, None), "aligned")
    _refused(f(P, P, P, P, P, P, P + 8, P, P, 0, 4, 8, 8, P, big, None), "aligned")


def test_gated_workspace_bytes(qglib):
    b = C.c_uint64()
    for M, N in ((1, 8), (16, 4096), (16, 4104), (65536, 1), (65537, 1), (4096, 8192), (1 << 29, 1 << 29)):
        assert qglib.qg_gemm_gated_backward_workspace_bytes(M, N, C.byref(b)) == 0
        assert pb.gemm_gated_backward_workspace_bytes(M, N) == b.value
    _refused(qglib.qg_gemm_gated_backward_workspace_bytes(0, 8, C.byref(b)), "workspace_bytes")
    with pytest.raises(ValueError):
        pb.gemm_gated_backward_workspace_bytes(4, 0)


def test_gated_dense_refuses_cpu_tensors(qglib):
    x, w = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((8, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16(x, w, w)
    with pytest.raises(ValueError):
        pb.gemm_gated_bf16_backward(x, x, w, w, x, x)
