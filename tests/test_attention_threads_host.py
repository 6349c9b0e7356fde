"""Calls of one rotation, cache or layer from several threads, without a GPU: each has its launches (made by one call of the
library, or by several for a layer's step) before the next one's begin, and close waits for the call that runs."""

import threading
import time
import types

import numpy as np
import pytest

from vesper_amd import _lib
from vesper_amd.attention import CachedAttention, HeadRotation, KVCache4, rotation_table
from vesper_amd.projections import FP8_LAYOUT


class Memory:
    """A device array of no device, which notes whether it is freed while a call runs."""

    def __init__(self, device):
        self.device, self.ptr = device, 1 << 20

    def __int__(self):
        return self.ptr

    def free(self):
        assert not self.device.running, "freed under a call"
        self.device.freed += 1


class Device:
    """A context and its library: calls take a while and note whom they met."""

    def __init__(self):
        self.lib, self.running, self.met, self.calls, self.freed = self, [], 0, [], 0
        self.cdll = _lib.load().cdll

    def _h(self):
        return None

    def empty(self, *_):
        return Memory(self)
    upload = empty

    def __getattr__(self, name):
        def call(*args):
            self.begin(threading.get_ident())
            time.sleep(0.01)
            self.running.remove(threading.get_ident())
            self.calls.append((threading.get_ident(), name))
        return call

    def begin(self, who):
        self.running.append(who)
        self.met += len(self.running) - 1


def in_threads(*calls):
    failures = []

    def one(call):
        try:
            call()
        except Exception as e:   # noqa: BLE001
            failures.append(e)
    threads = [threading.Thread(target=one, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
        assert not t.is_alive()
    return failures


def close_under(device, call, close):
    """close() while `call` runs in a thread; afterwards it is refused."""
    done = []
    thread = threading.Thread(target=lambda: done.append(in_threads(call)))
    thread.start()
    until = time.monotonic() + 20
    while not device.running and time.monotonic() < until:
        time.sleep(0.0005)
    close()
    thread.join(20)
    assert done == [[]]
    with pytest.raises(RuntimeError):
        call()


def test_a_cache_takes_one_attention_at_a_time():
    device = Device()
    cache = KVCache4(device, 4, 16, 1, 512, 512, query_heads=8, max_tokens=4, max_batch=4)
    attend = lambda: cache.attend_device(1 << 20, 2, 1 << 20, 1, 1 << 20, 2, 1 << 20, 1.0)  # noqa: E731
    append = lambda: cache.append_device(1 << 20, 1 << 20, 2)  # noqa: E731
    assert not in_threads(*[attend, append] * 4)
    assert device.met == 0 and len(device.calls) == 8
    close_under(device, attend, cache.close)
    assert device.freed == 3


def test_a_rotation_takes_one_call_at_a_time():
    device = Device()
    rot = HeadRotation(device, 64, norm=64)
    grad = rot.grad(1 << 20, 1, 1 << 20, 1 << 20, None, 1 << 20)
    assert not in_threads(*[lambda: rot.backward_device([grad], 3)] * 4, lambda: rot.apply_device([rot.set(1 << 20, 1, 1 << 20)], 3))
    assert device.met == 0 and len(device.calls) == 5
    assert rot.workspace is not None
    close_under(device, lambda: rot.backward_device([grad], 3), rot.close)
    assert device.freed == 1     # one workspace, whoever asked first


def test_a_layer_takes_one_step_at_a_time():
    device = Device()

    def project(name, x, tokens, y, stream=None):
        device.project()
    runtime = types.SimpleNamespace(ctx=device, block=32, has_wo_a=True, layout=dict(FP8_LAYOUT), project_device=project, _ready=lambda: None,
                                    tiled={"wo_a": 1 << 20}, lock=threading.Lock())
    layer = CachedAttention(runtime, 4, 16, rotation_table(8, 64), max_tokens=2, max_batch=2)
    device.calls.clear()
    step = lambda: layer.step_device(*[1 << 20, 2, 1 << 20, 1 << 20, 1 << 20, 1, 1 << 20, 2, 1 << 20])  # noqa: E731
    assert not in_threads(step, step, step)
    who = [w for w, _ in device.calls]
    assert device.met == 0 and sum(a != b for a, b in zip(who, who[1:])) == 2     # three steps, one behind the other
    each = len(who) // 3
    assert [n for _, n in device.calls[:each]] == [n for _, n in device.calls[-each:]]
    close_under(device, step, layer.close)
    assert len(device.calls) == 4 * each
