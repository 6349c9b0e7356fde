"""A scale is an FP32 number of the bank: what FP32 cannot hold is refused like infinity itself."""

import pytest

from tests.test_adapters_host import A, FakeContext
from vesper_amd.adapters import AdapterBank

LARGEST = 3.4028234663852886e38


@pytest.mark.parametrize("scale", [3.5e38, -3.5e38, 1e39, -1e300, float("inf"), float("nan")])
def test_a_scale_past_the_floats_is_refused(scale):
    bank = AdapterBank(FakeContext(), 64, 32, slots=4, max_rank=8, max_tokens=16)
    with pytest.raises(ValueError):
        bank.load_device(0, A, A, 8, scale)
    assert not bank.ctx.lib.calls


@pytest.mark.parametrize("scale", [LARGEST, -LARGEST, 1e-46, 0, 2])
def test_every_float_is_a_scale(scale):
    bank = AdapterBank(FakeContext(), 64, 32, slots=4, max_rank=8, max_tokens=16)
    bank.load_device(0, A, A, 8, scale)
    assert bank.ctx.lib.calls == ["adapters_load"]
