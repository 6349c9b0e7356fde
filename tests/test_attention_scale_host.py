"""Scales of logits whose product with log2(e) FP32 does not hold, without a GPU: refused, since zero logits would be NaN."""

import ctypes as C

import pytest

from vesper_amd import _lib

A = 1 << 20   # an aligned address that nothing reads


@pytest.mark.parametrize("scale,status", [(2.3e38, _lib.MX_ERR_STATE), (1e-45, _lib.MX_ERR_STATE), (2.4e38, _lib.MX_ERR_INVALID),
                                          (3.4e38, _lib.MX_ERR_INVALID), (0.0, _lib.MX_ERR_INVALID)])
def test_scales(scale, status):
    cache = _lib.MxKv4(A, A, A, A, 4, 16, 1, 128, 128)
    query = _lib.MxKv4Attend(A, 512, 4, 4, 2, None, A, 2, A, scale, 0, None, A, 512, None)
    assert _lib.load().cdll.mx_kv4_attend(C.c_void_p(0), C.byref(cache), C.byref(query), A, 1 << 40, None) == status
