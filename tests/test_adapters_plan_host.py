"""Plans that a bank of adapters cannot take, refused before any device work: a plan holds device addresses alone, so one
made for fewer groups would be read past its end, and one of other tokens would leave the output unwritten."""

import ctypes as C

import pytest

from tests.test_adapters_host import A, FakeContext, FakeLib
from vesper_amd import _lib
from vesper_amd.adapters import AdapterBank
from vesper_amd.dispatch import ExpertDispatch
from vesper_amd.projections import NativeProjections

T = 150   # tokens that take a plan


class PlanLib(FakeLib):
    """Keeps what plan the latest call had."""

    def adapters_apply(self, *args):
        self.calls.append("adapters_apply")
        self.plan = args[4]


class PlanContext(FakeContext):
    def __init__(self, ordinal=0):
        self.lib, self.ordinal = PlanLib(), ordinal

    def empty(self, shape, dtype):
        return _lib.DeviceArray(self, shape, dtype, A)


@pytest.fixture
def ctx():
    return PlanContext()


def bank_of(ctx, max_rank=8):
    return AdapterBank(ctx, 64, 32, slots=4, max_rank=max_rank, max_tokens=200)


def planned(ctx, experts=4, top_k=1, tokens=T):
    d = ExpertDispatch(ctx, experts, top_k, 200)
    d.plan_device(A, tokens)
    return d


def apply(bank, plan, tokens=T):
    bank.apply_device(A, A, tokens, A, A, plan=plan)


def test_a_plan_of_the_call_reaches_the_library(ctx):
    d = planned(ctx)
    for plan in (d, d.plan, _lib.MxRowPlan(A, A, A)):
        apply(bank_of(ctx), plan)
        assert ctx.lib.plan._obj.first == A
    apply(bank_of(ctx), None)
    assert ctx.lib.plan is None


@pytest.mark.parametrize("made", [{"experts": 3}, {"experts": 5}, {"top_k": 2}, {"tokens": T - 1}, {"tokens": T + 1},
                                  {"tokens": 0}])
@pytest.mark.parametrize("as_object", [True, False])
def test_a_plan_of_other_groups_or_tokens_is_refused(ctx, made, as_object):
    d, bank = planned(ctx, **made), bank_of(ctx)
    ctx.lib.calls.clear()
    with pytest.raises(ValueError):
        apply(bank, d if as_object else d.plan)
    assert not ctx.lib.calls


@pytest.mark.parametrize("max_rank,few", [(8, 128), (64, 128), (65, 64), (256, 64)])
def test_calls_of_few_tokens_leave_any_plan_unread(ctx, max_rank, few):
    bank, stale = bank_of(ctx, max_rank), planned(ctx, experts=2, tokens=7)
    for tokens in (1, few):
        apply(bank, stale, tokens)
        assert ctx.lib.plan is None
    with pytest.raises(ValueError):
        apply(bank, stale, few + 1)


def test_a_plan_that_is_not_there_is_refused(ctx):
    bank, d = bank_of(ctx), ExpertDispatch(ctx, 4, 1, 200)
    closed = planned(ctx)
    plan = closed.plan
    closed.close()
    ctx.lib.calls.clear()
    for none in (d, d.plan, closed, plan):   # nothing dispatched yet; its memory is gone
        with pytest.raises(RuntimeError):
            apply(bank, none)
    for wrong in (planned(PlanContext(1)), A, object()):   # another device's
        for tokens in (T,) if isinstance(wrong, ExpertDispatch) else (T, 3):
            with pytest.raises((ValueError, TypeError)):
                apply(bank, wrong, tokens)
    assert not ctx.lib.calls


def test_the_plan_follows_the_latest_dispatch(ctx):
    d, bank = planned(ctx), bank_of(ctx)
    plan = d.plan
    apply(bank, plan)
    d.plan_device(A, T + 7)
    with pytest.raises(ValueError):
        apply(bank, plan)
    apply(bank, plan, T + 7)


def test_a_projection_is_not_started_with_a_wrong_plan(ctx):
    """The adapters come after the projection in project_device; their refusal comes before it."""
    proj = NativeProjections.__new__(NativeProjections)
    proj.opened, proj.ctx, proj.layout, proj.block, proj.tiled = True, ctx, {"o": (64, 32)}, 32, {"o": A}
    proj.budget = type("Budget", (), {"acquire": lambda self, n: None})()
    proj.banks = {"o": bank_of(ctx)}
    wrong, right = planned(ctx, experts=3), planned(ctx)
    ctx.lib.calls.clear()
    for args in ({"plan": wrong}, {"plan": right, "tokens": T + 1}, {"tokens": 201}):
        with pytest.raises(ValueError):
            proj.project_device("o", A, args.get("tokens", T), A, adapters_ptr=A, plan=args.get("plan"))
    assert not ctx.lib.calls
    proj.project_device("o", A, T, A, adapters_ptr=A, plan=right)
    assert ctx.lib.calls == ["fp8_projection", "adapters_apply"]


def test_the_library_takes_the_plan_as_one(ctx):
    """The object that an ExpertDispatch gives stands for the C structure."""
    d = planned(ctx)
    assert isinstance(d.plan, _lib.MxRowPlan) and (d.plan.first, d.plan.pair_row, d.plan.row_pair) == (A, A, A)
    cdll = _lib.load().cdll
    assert cdll.mx_adapters_apply(None, A, 64, A, C.byref(d.plan), 4, A, 0, 64, A, 64, A, 1 << 30, None) == _lib.MX_ERR_STATE
