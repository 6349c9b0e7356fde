"""The hardware's rounding to BF16 against the software's, which the oracle's tests pin, on every FP32 bit pattern."""

import ctypes as C

import pytest

from vesper_amd import _lib

pytestmark = pytest.mark.gpu


def test_hardware_bf16_rounding_matches_on_every_float(gpu_ctx):
    mismatches = C.c_uint64(1)
    gpu_ctx.lib.check_bf16_pair(gpu_ctx._h(), C.byref(mismatches))
    assert mismatches.value == 0
    assert gpu_ctx.lib.cdll.mx_check_bf16_pair(gpu_ctx._h(), None) == _lib.MX_ERR_INVALID
