"""Gradients of two sets of heads whose dweight are one, without a GPU: refused, since either set's would be left there."""

import ctypes as C

import pytest

from vesper_amd import _lib

A = 1 << 20   # an aligned address that nothing reads


@pytest.mark.parametrize("first,second,status", [(A, A, _lib.MX_ERR_INVALID), (A, A + 508, _lib.MX_ERR_INVALID), (A + 4, A, _lib.MX_ERR_INVALID),
                                                 (A, A + 512, _lib.MX_ERR_STATE), (A + 512, A, _lib.MX_ERR_STATE), (A, None, _lib.MX_ERR_STATE),
                                                 (None, A, _lib.MX_ERR_STATE), (None, None, _lib.MX_ERR_STATE)])
def test_dweights(first, second, status):
    grads = (_lib.MxHeadsGrad * 2)(*(_lib.MxHeadsGrad(A, 1024, 8, None, A, 1024, A, 1024, w) for w in (first, second)))
    rotation = _lib.MxRotation(A, 16, A, 128, 128, 64, 64, 0, 0, 1e-6)
    cdll = _lib.load().cdll
    need = cdll.mx_rotate_heads_workspace_bytes(128)
    assert cdll.mx_rotate_heads_backward(C.c_void_p(0), grads, 2, 1, C.byref(rotation), 0, A, need, None) == status
