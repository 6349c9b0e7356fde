"""Numbers that do not fit the library's 32 bits, without a GPU: refused or, for a window, the same as the largest that does, and
never cut to another number."""

import ctypes as C

import pytest

from vesper_amd import _lib
from vesper_amd.attention import HeadRotation, KVCache4

A = 1 << 20


class Memory(int):
    ptr = A

    def free(self):
        pass


class Calls:
    """A context and library that keep the last attention call's query."""

    def __init__(self):
        self.lib, self.cdll, self.query = self, _lib.load().cdll, None

    def _h(self):
        return None

    def empty(self, *_):
        return Memory(A)

    def kv4_attend(self, handle, cache, query, *_):
        self.query = C.cast(query, C.POINTER(_lib.MxKv4Attend)).contents

    def __getattr__(self, name):
        return lambda *_: pytest.fail("a refused call reached the library")


@pytest.fixture
def calls():
    return Calls()


def cache_of(calls, **more):
    return KVCache4(calls, 4, 16, 1, 512, 512, **dict(dict(query_heads=8, max_tokens=4, max_batch=4), **more))


@pytest.mark.parametrize("window,taken", [(0, 0), (1, 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32, 2 ** 31 - 1),
                                          (2 ** 32 + 5, 2 ** 31 - 1), (2 ** 70, 2 ** 31 - 1)])
def test_windows_past_every_length(calls, window, taken):
    cache_of(calls).attend_device(A, 2, A, 1, A, 2, A, 1.0, window=window)
    assert calls.query.window == taken and calls.query.columns == 1


@pytest.mark.parametrize("change", [dict(window=-1), dict(window=-2 ** 32), dict(columns=2 ** 32 + 1), dict(columns=2 ** 26 + 1), dict(columns=-1),
                                    dict(tokens=2 ** 32 + 1), dict(batch=2 ** 32 + 1)])
def test_attention_refused(calls, change):
    args = dict(dict(q_ptr=A, tokens=2, table_ptr=A, columns=1, lengths_ptr=A, batch=2, out_ptr=A, scale=1.0), **change)
    with pytest.raises(ValueError):
        cache_of(calls).attend_device(**args)
    assert calls.query is None


@pytest.mark.parametrize("tokens", [-1, 2 ** 20 + 1, 2 ** 32, 2 ** 32 + 1])
def test_tokens_refused(calls, tokens):
    rot = HeadRotation(calls, 64, norm=64)
    for call in (lambda: cache_of(calls).append_device(A, A, tokens), lambda: rot.apply_device([rot.set(A, 1, A)], tokens),
                 lambda: rot.backward_device([rot.grad(A, 1, A, A)], tokens)):
        with pytest.raises(ValueError):
            call()


def test_heads_refused(calls):
    rot = HeadRotation(calls, 64)
    for heads in (-1, 2 ** 16 + 1, 2 ** 32 + 1):
        for make in (lambda: rot.set(A, heads, A), lambda: rot.grad(A, heads, A, A)):
            with pytest.raises(ValueError):
                make()
    with pytest.raises(ValueError):
        cache_of(calls, query_heads=2 ** 32 + 8)
