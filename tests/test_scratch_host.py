"""A context's scratch (mx_scratch.h, as the library compiles it): what a captured call was given is there until the context
closes, whatever grows it; without captures one buffer is held."""

import ctypes as C
from pathlib import Path

import numpy as np
import pytest

from vesper_amd import _lib

LIB = Path(__file__).resolve().parents[1] / "vesper_amd" / "libmxmoe_hostcheck.so"


def run(calls, failing=0):
    """[(status, buffer, its bytes, set of allocated buffers)] of calls (bytes, captured)."""
    assert LIB.exists(), "build first: python -m vesper_amd.build"
    fn = C.CDLL(str(LIB)).mxh_scratch
    fn.restype = C.c_int64
    size, captured = np.array([c[0] for c in calls], np.int64), np.array([c[1] for c in calls], np.int32)
    out = np.zeros((len(calls), 4), np.int64)
    left = fn(*(C.c_void_p(a.ctypes.data) for a in (size, captured)), len(calls), failing, C.c_void_p(out.ctypes.data))
    assert left == 0      # nothing outlives the context
    return [(int(s), int(p), int(b), {i for i in range(63) if live >> i & 1}) for s, p, b, live in out]


def test_without_captures_one_buffer_is_held():
    assert run([(4, 0), (3, 0), (9, 0), (9, 0), (10, 0)]) == [
        (0, 1, 4, {1}), (0, 1, 4, {1}), (0, 2, 9, {2}), (0, 2, 9, {2}), (0, 3, 10, {3})]


def test_what_a_capture_was_given_stays():
    got = run([(4, 0), (2, 1), (9, 0), (20, 0), (20, 1), (21, 0), (30, 0)])
    assert [g[1] for g in got] == [1, 1, 2, 3, 3, 4, 5]
    assert [g[3] for g in got] == [{1}, {1}, {1, 2}, {1, 3}, {1, 3}, {1, 3, 4}, {1, 3, 5}]


def test_nothing_is_released_while_a_stream_is_captured():
    assert [g[3] for g in run([(4, 0), (9, 1), (12, 1), (13, 0)])] == [{1}, {1, 2}, {1, 2, 3}, {1, 2, 3, 4}]


@pytest.mark.parametrize("captured", [0, 1])
def test_an_allocation_that_fails_leaves_what_captures_have(captured):
    got = run([(4, 1), (9, captured), (4, 0), (9, 0)], failing=2)
    assert got[1] == (-1, 1, 4, {1})
    assert got[2] == (0, 1, 4, {1}) and got[3] == (0, 3, 9, {1, 3})
    # without captures the old buffer has gone, and the next call allocates again
    assert run([(4, 0), (9, 0), (2, 0)], failing=2)[1:] == [(-1, 0, 0, set()), (0, 3, 2, {3})]


@pytest.mark.parametrize("shape", [(0, 128, 1), (32, 128, 1), (64, 64, 1), (64, 128, -1), (64, 128, 2 ** 20 + 1)])
def test_reserve_needs_a_context_first(shape):
    """A null context is refused before the shape is looked at, as by every FP8 call."""
    assert _lib.load().cdll.mx_fp8_reserve(None, *shape) == _lib.MX_ERR_STATE
