"""What a failing call and a failing close leave behind: nothing that is allocated, and no open context."""

import numpy as np
import pytest

from tests.test_gpu_projections import arrays_for
from vesper_amd import _lib
from vesper_amd.projections import NativeProjections
from vesper_amd.resources import MemoryBudget


class Lib:
    def __init__(self):
        self.cdll, self.fail_destroy = self, False

    def mx_adapters_workspace_bytes(self, *_):
        return 256

    def adapters_create(self, *args):
        args[-1]._obj.value = 0x10000

    def adapters_destroy(self, *_):
        if self.fail_destroy:
            raise _lib.HipError("destroy")

    def __getattr__(self, name):
        return lambda *args: None


class Context:
    """A context that counts its allocations and fails at the n-th from now on."""

    ordinal = 0

    def __init__(self):
        self.lib, self.live, self.next, self.left, self.closed = Lib(), set(), 0x1000, None, False

    def _h(self):
        return None

    def malloc(self, n):
        if self.left is not None:
            self.left -= 1
            if self.left < 0:
                raise MemoryError("cap")
        self.next += 0x1000
        self.live.add(self.next)
        return self.next

    def free(self, p):
        self.live.remove(p)

    def empty(self, shape, dtype):
        return _lib.DeviceArray(self, shape, dtype, self.malloc(1))

    def upload(self, a):
        return self.empty(a.shape, a.dtype)

    def download(self, ptr, shape, dtype, stream=None):
        return np.zeros(shape, dtype)

    def owned_bytes(self):
        return len(self.live), len(self.live)

    def close(self):
        self.closed = True


@pytest.fixture
def proj():
    layout = {"o": (64, 128)}
    p = NativeProjections(arrays_for(layout, 32, np.random.default_rng(0)), layout=layout)
    p.opened, p.ctx, p.tiled = True, Context(), {"o": 0x10000}
    p.budget = MemoryBudget(cap=1 << 30, available_floor=0, owner="test")
    p.budget.acquire(512 << 20)
    return p


@pytest.mark.parametrize("with_adapters", [False, True])
def test_fp8_frees_what_it_allocated_when_an_allocation_fails(proj, with_adapters):
    ids = None
    if with_adapters:
        proj.open_adapters("o", 2, 4, 8)
        ids = np.zeros(3, np.int32)
    values, before = np.zeros((3, 128), np.uint16), set(proj.ctx.live)
    for allowed in range(5 + with_adapters):
        proj.ctx.left = allowed
        with pytest.raises(MemoryError):
            proj.fp8("o", values, ids)
        assert proj.ctx.live == before, f"allocation {allowed + 1} failed"
    proj.ctx.left = None
    assert proj.fp8("o", values, ids)["output_bf16"].shape == (3, 64)
    assert proj.ctx.live == before


def test_the_context_closes_although_a_bank_does_not(proj):
    ctx = proj.ctx
    proj.open_adapters("o", 2, 4, 8)
    ctx.lib.fail_destroy = True
    with pytest.raises(_lib.HipError):
        proj.__exit__(None, None, None)
    assert ctx.closed and proj.ctx is None and not proj.banks and not proj.opened and not proj.tiled
    assert proj.budget.reserved == 0
