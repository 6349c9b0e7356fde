"""Calls of a rotation that is closed, or whose context is, without a GPU: RuntimeError before anything else, as of a closed
cache."""

import types

import numpy as np
import pytest

from vesper_amd import _lib
from vesper_amd.attention import HeadRotation


def opened():
    """A rotation of a context that gives nothing but the library and a handle."""
    ctx = types.SimpleNamespace(lib=_lib.load(), _h=lambda: 1)
    return HeadRotation(ctx, 64, norm=64)


CALLS = [lambda r: r.apply(np.zeros((2, 1, 64), np.uint16)), lambda r: r.backward(*[np.zeros((2, 1, 64), np.float32)] * 2),
         lambda r: r.apply_device([], 1), lambda r: r.backward_device([], 1), lambda r: r.open_gradients(), lambda r: r.struct()]


@pytest.mark.parametrize("call", CALLS)
def test_closed_rotations(call):
    rot = opened()
    rot.close()
    rot.close()
    with pytest.raises(RuntimeError, match="closed"):
        call(rot)


@pytest.mark.parametrize("call", CALLS)
def test_rotations_of_closed_contexts(call):
    rot = opened()

    def closed():
        raise RuntimeError("device context is closed")
    rot.ctx._h = closed
    with pytest.raises(RuntimeError, match="closed"):
        call(rot)
