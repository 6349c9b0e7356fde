"""Tokens by expert and back without a GPU: the oracle's own properties, and every refusal that comes before device
work (through the library, whose argument checks need no device, and through ExpertDispatch)."""

import ctypes as C

import numpy as np
import pytest

from oracle import dispatch as oracle
from vesper_amd import _lib
from vesper_amd.dispatch import ExpertDispatch, host_rows, row_type
from vesper_amd.moe import participation


def test_plan_is_participations_order():
    rng = np.random.default_rng(1)
    ids = np.stack([rng.permutation(12)[:3] for _ in range(9)]).astype(np.int32)
    first, pair_row, row_pair = oracle.plan(ids, 12)
    selected = participation(ids, experts=12, top_k=3)
    for e in range(12):
        tokens = row_pair[first[e]:first[e + 1]] // 3
        np.testing.assert_array_equal(tokens, selected.get(e, []))
    assert sorted(pair_row.reshape(-1)) == list(range(27))


def test_pairs_of_absent_experts_come_last_and_have_no_row():
    first, pair_row, row_pair = oracle.plan([[4, -1], [0, 4], [7, 0]], 5)
    np.testing.assert_array_equal(first, [0, 2, 2, 2, 2, 4])
    np.testing.assert_array_equal(pair_row, [[2, -1], [0, 3], [-1, 1]])
    np.testing.assert_array_equal(row_pair, [2, 5, 0, 3, 1, 4])


def test_gradients_of_the_oracle_against_differences():
    rng = np.random.default_rng(2)
    ids = np.array([[1, 0], [2, 9], [0, 0]])
    _, pair_row, _ = oracle.plan(ids, 3)
    rows, weights, dy = rng.standard_normal((6, 4)), rng.standard_normal((3, 2)), rng.standard_normal((3, 4))
    drows, dweights, _ = oracle.combine_backward(dy, rows, pair_row, weights)
    loss = lambda: float((oracle.combine(rows, pair_row, weights)[0] * dy).sum())  # noqa: E731
    step = 1e-6
    for array, grad in ((rows, drows), (weights, dweights)):
        for index in np.ndindex(array.shape):
            kept = array[index]
            array[index] = kept + step
            up = loss()
            array[index] = kept - step
            down = loss()
            array[index] = kept
            # a loss linear in each entry: the quotient is off by the sums' rounding over the step alone
            assert abs((up - down) / (2 * step) - grad[index]) < 1e-7


A, B = 0x10000, 0x20000   # addresses that no check follows


def plan_at(first=A, pair_row=A, row_pair=A):
    return C.byref(_lib.MxRowPlan(first, pair_row, row_pair))


def status(name, *args):
    return getattr(_lib.load().cdll, "mx_" + name)(*args)


def dispatch_args(**changed):
    args = dict(ctx=None, ids=A, tokens=4, top_k=2, groups=8, plan=plan_at(), x=A, dtype=0, width=64, weights=None,
                rows=2 * A, row_weights=None, stream=None)
    args.update(changed)
    return list(args.values())


@pytest.mark.parametrize("changed", [
    {"tokens": -1}, {"tokens": (1 << 18) + 1}, {"top_k": 0}, {"top_k": 33}, {"groups": 0}, {"groups": 1025},
    {"plan": None}, {"plan": plan_at(first=None)}, {"plan": plan_at(pair_row=None)}, {"plan": plan_at(row_pair=None)},
    {"plan": plan_at(row_pair=A + 2)}, {"x": None}, {"rows": None}, {"ids": None, "x": None, "rows": None},
    {"weights": A}, {"row_weights": A}, {"x": None, "rows": None, "weights": A, "row_weights": A},
    {"dtype": 3}, {"dtype": -1}, {"width": 0}, {"width": -5}, {"width": (1 << 24) + 1}, {"x": A + 1},
    {"rows": A + 1}, {"rows": A}, {"dtype": 1, "x": A + 2}, {"ids": A + 2}, {"weights": A + 1, "row_weights": A},
])
def test_dispatch_refusals(changed):
    assert status("dispatch", *dispatch_args(**changed)) == _lib.MX_ERR_INVALID


def test_valid_arguments_reach_the_context_check():
    """The refusals above are the arguments': the same calls with valid ones stop at the missing context."""
    for changed in ({}, {"tokens": 0}, {"x": None, "rows": None}, {"ids": None}, {"dtype": 2, "x": A + 1},
                    {"weights": A, "row_weights": A}):
        assert status("dispatch", *dispatch_args(**changed)) == _lib.MX_ERR_STATE
    assert status("combine", None, A, 0, A, None, 2 * A, 4, 2, 64, 2 * A, None) == _lib.MX_ERR_STATE
    assert status("combine_backward", None, 2 * A, A, 0, A, None, 4, 2, 64, A, A, None) == _lib.MX_ERR_STATE
    assert status("dispatch_backward", None, A, 0, A, None, 4, 2, 64, 2 * A, None, None) == _lib.MX_ERR_STATE


def test_outputs_that_are_an_input_are_refused():
    """Rows change places between these: what is read would be another row's result."""
    assert status("combine", None, A, 0, A, None, None, 4, 2, 64, A, None) == _lib.MX_ERR_INVALID
    assert status("combine_backward", None, A, 2 * A, 0, A, None, 4, 1, 64, A, A, None) == _lib.MX_ERR_INVALID
    assert status("dispatch_backward", None, A, 0, A, None, 4, 2, 64, A, None, None) == _lib.MX_ERR_INVALID


@pytest.mark.parametrize("args", [
    (None, 0, A, None, None, 4, 2, 64, B), (A, 0, None, None, None, 4, 2, 64, B), (A, 0, A, None, None, 4, 2, 64, None),
    (A, 2, A, None, None, 4, 2, 64, B), (A, 0, A, None, None, -1, 2, 64, B), (A, 0, A, None, None, 4, 40, 64, B),
    (A, 0, A, None, None, 4, 2, 0, B), (A + 1, 0, A, None, None, 4, 2, 64, B), (A, 1, A, None, A + 2, 4, 2, 64, B),
    (A, 0, A + 2, None, None, 4, 2, 64, B), (A, 0, A, A + 1, None, 4, 2, 64, B),
])
def test_combine_refusals(args):
    assert status("combine", None, *args, None) == _lib.MX_ERR_INVALID


@pytest.mark.parametrize("args", [
    (None, A, 0, A, None, 4, 2, 64, B, A), (A, None, 0, A, None, 4, 2, 64, B, A), (A, A, 0, None, None, 4, 2, 64, B, A),
    (A, A, 0, A, None, 4, 2, 64, None, None), (A, A, 2, A, None, 4, 2, 64, B, A), (A, A, 0, A, None, 4, 0, 64, B, A),
    (A, A, 0, A, None, 4, 2, -1, B, A), (A, A, 1, A, None, 4, 2, 64, A + 2, A), (A, A, 0, A, None, 4, 2, 64, B, A + 2),
])
def test_combine_backward_refusals(args):
    assert status("combine_backward", None, *args, None) == _lib.MX_ERR_INVALID


@pytest.mark.parametrize("args", [
    (None, 0, A, None, 4, 2, 64, B, None), (A, 0, None, None, 4, 2, 64, B, None), (A, 0, A, None, 4, 2, 64, None, None),
    (A, 0, A, A, 4, 2, 64, B, None), (A, 0, A, None, 4, 2, 64, B, A), (A, 2, A, None, 4, 2, 64, B, None),
    (A, 0, A, None, 1 << 20, 2, 64, B, None), (A + 1, 0, A, None, 4, 2, 64, B, None),
])
def test_dispatch_backward_refusals(args):
    assert status("dispatch_backward", None, *args, None) == _lib.MX_ERR_INVALID


class FakeContext:
    """A context whose allocations are host numbers: the refusals below must come before any library call."""

    def empty(self, shape, dtype):
        return _lib.DeviceArray(self, shape, dtype, A)

    def free(self, p):
        pass

    @property
    def lib(self):
        raise AssertionError("device work before the refusal")


@pytest.mark.parametrize("args", [(0, 2, 4), (1025, 2, 4), (8, 0, 4), (8, 33, 4), (8, 2, 0), (8, 2, (1 << 18) + 1)])
def test_expert_dispatch_refuses_its_sizes(args):
    with pytest.raises(ValueError):
        ExpertDispatch(FakeContext(), *args)


def test_expert_dispatch_refuses_before_device_work():
    d = ExpertDispatch(FakeContext(), 8, 2, 4)
    x = np.zeros((3, 64), np.uint16)
    ids = np.zeros((3, 2), np.int32)
    for bad_ids, bad_x in ((ids.astype(np.float32), x), (ids[:, :1], x), (ids, x[:2]), (ids, x.astype(np.float64)),
                           (ids, x[0]), (np.zeros((5, 2), np.int32), np.zeros((5, 64), np.uint16)),
                           (np.full((3, 2), 2 ** 31, np.int64), x)):
        with pytest.raises(ValueError):
            d.dispatch(bad_ids, bad_x)
    with pytest.raises(ValueError):
        d.dispatch(ids, x, np.zeros((3, 3)))
    with pytest.raises(RuntimeError):   # nothing dispatched yet
        d.combine(np.zeros((6, 64), np.uint16))
    with pytest.raises(ValueError):
        d.dispatch_device(A, 5, A, 64, A)
    d.tokens = 3
    rows = np.zeros((6, 64), np.uint16)
    for call in (lambda: d.combine(rows[:5]), lambda: d.combine(rows.astype(np.uint8)),
                 lambda: d.combine(rows, np.zeros((2, 2))), lambda: d.combine(rows, None, x.astype(np.float32)),
                 lambda: d.combine(rows, None, x[:, :32]), lambda: d.combine_backward(x, rows[:, :32]),
                 lambda: d.combine_backward(x, rows.astype(np.float32)), lambda: d.dispatch_backward(rows[:4]),
                 lambda: d.dispatch_backward(rows, np.zeros(5)), lambda: d.move_device(A, 64, A, "f64"),
                 lambda: d.combine_device(A, 64, A, "u8")):
        with pytest.raises(ValueError):
            call()
    d.close()
    with pytest.raises(RuntimeError):
        d.combine(rows)


def test_row_types():
    assert (row_type("bf16"), row_type("f32"), row_type("u8", True)) == (0, 1, 2)
    assert host_rows(np.zeros((2, 3), np.float32))[1] == "f32"
    for bad in ("u8", "fp16", ""):
        with pytest.raises(ValueError):
            row_type(bad)
