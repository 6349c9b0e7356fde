"""Low-rank adapters without a GPU: the oracle against one dense matrix, and every refusal before device work."""

import ctypes as C

import numpy as np
import pytest

from oracle import adapters as oracle
from vesper_amd import _lib
from vesper_amd.adapters import AdapterBank

A = 0x10000


def test_oracle_is_the_dense_update():
    rng = np.random.default_rng(0)
    down, up = rng.standard_normal((3, 16)), rng.standard_normal((8, 3))
    x, base = rng.standard_normal((4, 16)), rng.standard_normal((4, 8))
    y, size = oracle.apply(x, [1, -1, 0, 1], base, {1: (down, up, 0.5)})
    dense = base + 0.5 * x @ (up @ down).T
    np.testing.assert_allclose(y[[0, 3]], dense[[0, 3]], rtol=1e-12)
    np.testing.assert_array_equal(y[[1, 2]], base[[1, 2]])
    assert (size >= np.abs(y)).all()


@pytest.mark.parametrize("args", [(0, 64, 4, 8), (12, 64, 4, 8), (64, 0, 4, 8), (64, 60, 4, 8), (64, (1 << 20) + 8, 4, 8),
                                  (64, 64, 0, 8), (64, 64, 1025, 8), (64, 64, 4, 0), (64, 64, 4, 257)])
def test_bank_sizes(args):
    out = C.c_void_p()
    cdll = _lib.load().cdll
    assert cdll.mx_adapters_create(None, *args, C.byref(out)) == _lib.MX_ERR_INVALID
    assert cdll.mx_adapters_create(None, 64, 64, 4, 8, None) == _lib.MX_ERR_INVALID
    with pytest.raises(ValueError):
        AdapterBank(None, *args, 16)
    with pytest.raises(ValueError):
        AdapterBank(None, 64, 64, 4, 8, 0)


def test_valid_sizes_reach_the_context_and_a_closed_bank_is_a_state_error():
    out = C.c_void_p()
    cdll = _lib.load().cdll
    assert cdll.mx_adapters_create(None, 64, 64, 4, 8, C.byref(out)) == _lib.MX_ERR_STATE and not out
    assert cdll.mx_adapters_load(None, 0, A, A, 8, 1.0, None) == _lib.MX_ERR_STATE
    assert cdll.mx_adapters_apply(None, A, 64, A, None, 4, A, 0, 64, A, 64, A, 1 << 30, None) == _lib.MX_ERR_STATE
    assert cdll.mx_adapters_workspace_bytes(None, 4) == 0
    assert cdll.mx_adapters_destroy(None) == _lib.MX_OK


class FakeLib:
    """Stands for the library of an open bank: whatever reaches it is counted."""

    def __init__(self):
        self.calls = []
        self.cdll = self

    def mx_adapters_workspace_bytes(self, *_):
        return 256

    def adapters_create(self, *args):
        args[-1]._obj.value = A

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name)


class FakeContext:
    def __init__(self):
        self.lib = FakeLib()

    def _h(self):
        return None

    def malloc(self, n):
        return A

    def free(self, p):
        pass

    def upload(self, a):
        raise AssertionError("device work before the refusal")


@pytest.fixture
def bank():
    return AdapterBank(FakeContext(), 64, 32, slots=4, max_rank=8, max_tokens=16)


def test_load_refusals(bank):
    down, up = np.zeros((8, 32), np.uint16), np.zeros((64, 8), np.uint16)
    nan = down.copy()
    nan[0, 0] = 0x7FC0
    for args in ((4, down, up), (-1, down, up), (True, down, up), (0, down[:, :16], up), (0, down, up[:, :4]),
                 (0, down.astype(np.float32), up), (0, nan, up), (0, down, up, np.inf), (0, np.zeros((0, 32), np.uint16), up),
                 (0, np.zeros((9, 32), np.uint16), np.zeros((64, 9), np.uint16)), (0, down[0], up)):
        with pytest.raises(ValueError):
            bank.load(*args)
    for args in ((4, A, A, 8), (0, A, A, 0), (0, A, A, 9), (0, A, A, 8, np.nan)):
        with pytest.raises(ValueError):
            bank.load_device(*args)
    with pytest.raises(ValueError):
        bank.clear(4)
    assert not bank.ctx.lib.calls


def test_apply_refusals(bank):
    x, ids, base = np.zeros((3, 32), np.uint16), np.zeros(3, np.int32), np.zeros((3, 64), np.uint16)
    inf = x.copy()
    inf[1, 1] = 0x7F80
    for args in ((x[:, :16], ids, base), (x[0], ids, base), (inf, ids, base), (x.astype(np.float32), ids, base),
                 (x, ids[:2], base), (x, ids.astype(np.float32), base), (x, ids + 4, base), (x, ids - 2, base),
                 (x, ids, base[:, :32]), (x, ids, base.astype(np.float64)),
                 (np.zeros((17, 32), np.uint16), np.zeros(17, np.int32), np.zeros((17, 64), np.uint16))):
        with pytest.raises(ValueError):
            bank.apply(*args)
    for args in ((A, A, 17, A, A), (A, A, -1, A, A), (A, A, 3, A, A, "u8")):
        with pytest.raises(ValueError):
            bank.apply_device(*args)
    assert not bank.ctx.lib.calls
    bank.close()
    for call in (lambda: bank.apply(x, ids, base), lambda: bank.apply_device(A, A, 3, A, A), lambda: bank.clear(0)):
        with pytest.raises(RuntimeError):
            call()


def test_a_closed_context_has_taken_the_bank(bank):
    """No call hands the library a bank whose context is gone."""
    def closed():
        raise RuntimeError("device context is closed")
    bank.ctx._h = closed
    for call in (lambda: bank.apply_device(A, A, 3, A, A), lambda: bank.load_device(0, A, A, 8), lambda: bank.clear(0),
                 bank.close):
        with pytest.raises(RuntimeError):
            call()
    assert not bank.ctx.lib.calls
