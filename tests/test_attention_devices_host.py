"""A rotation of another device than the cache's, without a GPU: refused before the library is called."""

import pytest

from tests.test_attention_numbers_host import A, Calls
from vesper_amd.attention import HeadRotation, KVCache4, rotation_table


class Device(Calls):
    def __init__(self, ordinal):
        super().__init__()
        self.ordinal, self.appended = ordinal, 0

    def upload(self, *_):
        return self.empty()

    def kv4_append(self, *_):
        self.appended += 1


def test_rotations_of_another_device():
    here, there = Device(0), Device(1)
    cache = KVCache4(here, 4, 16, 1, 512, 512, query_heads=8, max_tokens=4, max_batch=4)
    rotations = [HeadRotation(d, 512, norm=512, dims=64, table=rotation_table(8, 64)) for d in (here, Device(0), there)]
    for rot in rotations[:2]:     # another context of the same device will do
        cache.append_device(A, A, 2, rotation=rot, positions_ptr=A)
    assert here.appended == 2
    with pytest.raises(ValueError, match="device 1"):
        cache.append_device(A, A, 2, rotation=rotations[2], positions_ptr=A)
    assert here.appended == 2
