"""The library's own refusal of a scale that is no finite number."""

import pytest

from vesper_amd import _lib
from vesper_amd.adapters import AdapterBank

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan"), 1e39])
def test_load_refuses_a_scale_that_is_not_finite(gpu_ctx, scale):
    with AdapterBank(gpu_ctx, 64, 32, 2, 8, 4) as bank:
        a = 1 << 20   # an address that no check follows
        load = gpu_ctx.lib.cdll.mx_adapters_load
        assert load(bank.handle, 0, a, a, 8, scale, None) == _lib.MX_ERR_INVALID
        assert load(bank.handle, 0, None, None, 0, 0.0, None) == _lib.MX_OK
