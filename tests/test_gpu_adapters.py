"""Low-rank adapters on the device against the 64-bit oracle.

On small integers every product, sum and term is exact, so results are the oracle's rounded once, bit for bit. On random
values: an FP32 chain of n additions is within n 2^-24 of the terms' magnitudes, here at most width / 32 + rank / 16 + 50
matrix steps and additions, counted twice for what a matrix step rounds inside; h as two BF16 terms is within 2^-8 2^-8 =
2^-16 of its value; the result's rounding is half a BF16 step, 2^-8 of its value.
"""

import ctypes as C

import numpy as np
import pytest

from oracle import adapters as oracle
from oracle.formats import bf16_bits, bf16_values
from tests.test_gpu_projections import arrays_for
from tests.test_gpu_scratch import Graph
from vesper_amd import _lib
from vesper_amd.adapters import AdapterBank
from vesper_amd.dispatch import ExpertDispatch
from vesper_amd.projections import NativeProjections

pytestmark = pytest.mark.gpu

RANKS = (1, 16, 7, 64, 17, 33, 100, 256)


def integers(rng, lo, hi, shape):
    return rng.integers(lo, hi + 1, shape).astype(np.float32)


def adapter(rng, rows, width, rank, exact):
    """(down, up, scale) values that BF16 holds."""
    if exact:
        return integers(rng, -2, 2, (rank, width)), integers(rng, -2, 2, (rows, rank)), float(rng.choice([0.5, 1, -2]))
    down = bf16_values(bf16_bits(rng.standard_normal((rank, width)).astype(np.float32)))
    up = bf16_values(bf16_bits((rng.standard_normal((rows, rank)) / np.sqrt(width * rank)).astype(np.float32)))
    return down, up, float(rng.uniform(0.5, 2))


def fill(bank, rng, adapters):
    for slot, (down, up, scale) in adapters.items():
        bank.load(slot, bf16_bits(down), bf16_bits(up), scale)


def inputs(rng, tokens, rows, width, exact, dtype):
    x = integers(rng, -2, 2, (tokens, width)) if exact else rng.standard_normal((tokens, width)).astype(np.float32)
    base = integers(rng, -99, 99, (tokens, rows)) if exact else rng.standard_normal((tokens, rows)).astype(np.float32)
    return bf16_bits(x), base if dtype == "f32" else bf16_bits(base)


def values(a):
    return bf16_values(a) if a.dtype == np.uint16 else a


def check(got, x, ids, base, adapters, exact):
    want, size = oracle.apply(values(x), ids, values(base), adapters)
    if exact:
        # every partial sum is a multiple of 1/2 below 2^23 (x, down, up at most 2, width 1600, rank 256, scale 2)
        np.testing.assert_array_equal(got, bf16_bits(want.astype(np.float32)))
        return
    rank = max([a[0].shape[0] for a in adapters.values()], default=0)
    steps = x.shape[1] / 32 + rank / 16 + 50
    limit = np.abs(want) * 2.0 ** -8 + (1 + 2.0 ** -8) * size * (2.0 ** -16 + 2 * steps * 2.0 ** -24)
    worst = np.max(np.abs(values(got).astype(np.float64) - want) - limit)
    assert worst <= 0, f"{worst:.3e} past the limit"


# (tokens, rows, width, slots, max_rank): either form and its border, ragged tiles, one value more than a chunk or block
SHAPES = [(1, 8, 8, 1, 1), (1, 64, 32, 1, 16), (1, 2112, 1536, 3, 64), (2, 72, 40, 2, 7), (5, 24, 520, 8, 256),
          (31, 576, 128, 5, 17), (32, 136, 1600, 4, 33), (33, 64, 72, 3, 16), (40, 1032, 2048, 2, 32), (47, 200, 264, 8, 256), (60, 24, 104, 1, 128),
          (64, 1024, 96, 70, 64), (65, 8, 1536, 1, 100), (100, 320, 8, 90, 8), (127, 72, 1032, 3, 40), (128, 136, 328, 40, 16), (129, 64, 96, 5, 64),
          (257, 88, 160, 6, 64),
          (150, 136, 600, 8, 256), (1000, 264, 520, 8, 128)]


@pytest.mark.parametrize("tokens,rows,width,slots,max_rank", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("exact", [True, False])
def test_apply(gpu_ctx, tokens, rows, width, slots, max_rank, dtype, exact):
    rng = np.random.default_rng(tokens * 7 + rows)
    with AdapterBank(gpu_ctx, rows, width, slots, max_rank, tokens) as bank:
        # every third slot stays empty; ranks of their own, the largest in slot 0
        adapters = {s: adapter(rng, rows, width, max_rank if s == 0 else min(max_rank, RANKS[s % len(RANKS)]), exact)
                    for s in range(slots) if s % 3 != 2}
        fill(bank, rng, adapters)
        x, base = inputs(rng, tokens, rows, width, exact, dtype)
        ids = rng.integers(-1, slots, tokens).astype(np.int32)
        if tokens == 1:
            ids[0] = 0
        check(bank.apply(x, ids, base), x, ids, base, adapters, exact)


@pytest.mark.parametrize("tokens", [4, 17, 64, 90, 128, 150])
def test_all_or_no_tokens_of_one_adapter(gpu_ctx, tokens):
    rng = np.random.default_rng(tokens)
    rows, width = 72, 136
    with AdapterBank(gpu_ctx, rows, width, 4, 24, tokens) as bank:
        adapters = {1: adapter(rng, rows, width, 24, True)}
        fill(bank, rng, adapters)
        x, base = inputs(rng, tokens, rows, width, True, "bf16")
        base[0, :3] = (0x8000, 0x7F80, 0x7FC0)   # -0, infinity, NaN pass through where there is no adapter
        for slot in (1, 0, -1):
            ids = np.full(tokens, slot, np.int32)
            got = bank.apply(x, ids, base)
            if slot == 1:
                check(got[1:], x[1:], ids[1:], base[1:], adapters, True)
                assert got[0, 1] == 0x7F80 and np.isnan(bf16_values(got[0, 2:3]))[0]
            else:
                np.testing.assert_array_equal(got, base)
        assert bank.apply(x[:0], ids[:0], base[:0]).shape == (0, rows)


@pytest.mark.parametrize("tokens", [3, 70, 170])
def test_strided_rows_in_place_with_and_without_a_plan(gpu_ctx, tokens):
    """The columns of a stacked output (two projections of one input), in place; what lies beside them stays."""
    rng = np.random.default_rng(tokens)
    rows, width, stride, column, x_stride = 72, 40, 120, 16, 56
    adapters = {s: adapter(rng, rows, width, 1 + 5 * s, True) for s in range(4)}
    ids = rng.integers(-1, 6, tokens).astype(np.int32)   # on the device, ids past the slots are tokens without one
    x = bf16_bits(integers(rng, -2, 2, (tokens, x_stride)))
    x[:, width:] = 0x7FC0                                # never read
    stacked = bf16_bits(integers(rng, -99, 99, (tokens, stride)))
    base = stacked[:, column:column + rows]
    with AdapterBank(gpu_ctx, rows, width, 4, 16, tokens) as bank, ExpertDispatch(gpu_ctx, 4, 1, tokens) as d:
        fill(bank, rng, adapters)
        xd, idd, yd = (gpu_ctx.upload(a) for a in (x, ids, stacked))
        d.plan_device(idd, tokens)
        for plan in (None, d.plan):
            yd.upload(stacked)
            at = yd.ptr + 2 * column
            bank.apply_device(xd, idd, tokens, at, at, x_stride=x_stride, base_stride=stride, y_stride=stride, plan=plan)
            got = yd.download()
            check(got[:, column:column + rows], x[:, :width], ids, base, adapters, True)
            got[:, column:column + rows] = base
            np.testing.assert_array_equal(got, stacked)
        for a in (xd, idd, yd):
            a.free()


def test_infinite_and_nan_inputs_stay_with_their_token(gpu_ctx):
    rng = np.random.default_rng(0)
    rows, width = 64, 64
    for tokens in (3, 40, 140):
        adapters = {0: adapter(rng, rows, width, 5, True)}
        with AdapterBank(gpu_ctx, rows, width, 1, 16, tokens) as bank:
            fill(bank, rng, adapters)
            x, base = inputs(rng, tokens, rows, width, True, "f32")
            spoiled = x.copy()
            spoiled[1] = 0x7FC0
            dev = [gpu_ctx.upload(a) for a in (spoiled, np.zeros(tokens, np.int32), base, np.zeros((tokens, rows), np.uint16))]
            bank.apply_device(dev[0], dev[1], tokens, dev[2], dev[3], "f32")
            got = dev[3].download()
            keep = np.arange(tokens) != 1
            check(got[keep], x[keep], np.zeros(tokens - 1, int), base[keep], adapters, True)
            # where up's row is not zero, NaN reaches the result
            assert np.isnan(bf16_values(got[1]))[np.abs(adapters[0][1]).sum(1) > 0].all()
            for a in dev:
                a.free()


def test_slots_are_replaced_and_emptied(gpu_ctx):
    rng = np.random.default_rng(6)
    rows, width, tokens = 40, 72, 150
    x, base = inputs(rng, tokens, rows, width, True, "f32")
    ids = rng.integers(0, 2, tokens).astype(np.int32)
    with AdapterBank(gpu_ctx, rows, width, 2, 40, tokens) as bank:
        adapters = {}
        for step, rank in enumerate((40, 3, 20)):   # a smaller rank after a larger: nothing of the larger is left
            adapters[step % 2] = adapter(rng, rows, width, rank, True)
            adapters[0] = adapter(rng, rows, width, rank, True)
            fill(bank, rng, adapters)
            check(bank.apply(x, ids, base), x, ids, base, adapters, True)
        bank.clear(0)
        del adapters[0]
        check(bank.apply(x, ids, base), x, ids, base, adapters, True)


def test_the_result_does_not_depend_on_the_tokens_order(gpu_ctx):
    """A call's tokens in any order, and the same call again, give the same bits."""
    rng = np.random.default_rng(14)
    rows, width = 200, 1024
    for tokens in (20, 100, 300):
        with AdapterBank(gpu_ctx, rows, width, 5, 32, tokens) as bank:
            fill(bank, rng, {s: adapter(rng, rows, width, 32 - 3 * s, False) for s in range(5)})
            x, base = inputs(rng, tokens, rows, width, False, "bf16")
            ids = rng.integers(-1, 5, tokens).astype(np.int32)
            y = bank.apply(x, ids, base)
            order = rng.permutation(tokens)
            np.testing.assert_array_equal(bank.apply(x[order], ids[order], base[order]), y[order])
            np.testing.assert_array_equal(bank.apply(x, ids, base), y)


@pytest.mark.parametrize("tokens,seed", [(6, 0), (120, 1), (200, 2)])
def test_captured_calls_replay_on_new_inputs(tokens, seed):
    rows, width, slots = 136, 96, 3
    rng = np.random.default_rng(seed)
    with _lib.Context(0) as ctx, AdapterBank(ctx, rows, width, slots, 16, tokens) as bank:
        adapters = {s: adapter(rng, rows, width, 16, True) for s in range(slots)}
        fill(bank, rng, adapters)
        stream = ctx.stream()
        x, base = inputs(rng, tokens, rows, width, True, "f32")
        xd, idd, bd, yd = (ctx.upload(a) for a in (x, np.zeros(tokens, np.int32), base, np.zeros((tokens, rows), np.uint16)))
        graph = Graph(ctx, stream, lambda: bank.apply_device(xd, idd, tokens, bd, yd, "f32", stream=stream))
        for _ in range(4):
            x, base = inputs(rng, tokens, rows, width, True, "f32")
            ids = rng.integers(-1, slots, tokens).astype(np.int32)
            for dev, host in ((xd, x), (idd, ids), (bd, base)):
                dev.upload(host)
            ctx.sync()
            graph.launch()
            check(yd.download(), x, ids, base, adapters, True)
            bank.apply(x, ids[::-1].copy(), base)   # the program's own call between replays, on the same workspace
        graph.close()
        for a in (xd, idd, bd, yd):
            a.free()
        ctx.destroy_stream(stream)


@pytest.mark.parametrize("tokens", [100, 300])
def test_rows_past_32_bits(gpu_ctx, tokens):
    """Strides that put the last rows more than 2^31 values (and for the grouped form 2^32) from the first."""
    rng = np.random.default_rng(tokens)
    rows, width, stride = 72, 104, 1 << 25
    adapters = {s: adapter(rng, rows, width, 9 + s, True) for s in range(2)}
    ids = rng.integers(-1, 2, tokens).astype(np.int32)
    x, base = inputs(rng, tokens, rows, width, True, "bf16")
    with AdapterBank(gpu_ctx, rows, width, 2, 16, tokens) as bank:
        fill(bank, rng, adapters)
        at = gpu_ctx.malloc(2 * stride * tokens)   # a row's x, and 256 bytes on its base, which y replaces
        idd = gpu_ctx.upload(ids)
        for t in range(tokens):
            gpu_ctx.copy_h2d(at + 2 * stride * t, x[t])
            gpu_ctx.copy_h2d(at + 2 * stride * t + 256, base[t])
        bank.apply_device(at, idd, tokens, at + 256, at + 256, x_stride=stride, base_stride=stride, y_stride=stride)
        got = np.stack([gpu_ctx.download(at + 2 * stride * t + 256, (rows,), np.uint16) for t in range(tokens)])
        check(got, x, ids, base, adapters, True)
        idd.free()
        gpu_ctx.free(at)


def test_calls_larger_than_the_caches(gpu_ctx):
    """x and y of more than 96 MiB; 1600 of the columns of x are not zero, which keeps every sum exact."""
    rng = np.random.default_rng(9)
    tokens, rows, width, slots = 7100, 3592, 7176, 3
    adapters = {s: adapter(rng, rows, width, 16 - 5 * s, True) for s in range(slots)}
    ids = rng.integers(-1, slots, tokens).astype(np.int32)
    x, base = inputs(rng, tokens, rows, width, True, "bf16")
    x[:, rng.permutation(width)[1600:]] = 0
    with AdapterBank(gpu_ctx, rows, width, slots, 16, tokens) as bank:
        fill(bank, rng, adapters)
        check(bank.apply(x, ids, base), x, ids, base, adapters, True)


@pytest.mark.parametrize("first", [[0, 60, 40, 170], [0, 30, 60, 171], [0, -1, 60, 170], [1, 30, 60, 170], [170] * 4,
                                   [0, 1 << 30, 1 << 30, 170]])
def test_a_plan_that_is_none_does_nothing(gpu_ctx, first):
    """Groups that do not cover the tokens in order: y is left as it was, and nothing out of range is touched. The same
    call by a right plan follows."""
    rng = np.random.default_rng(1)
    tokens, rows, width, slots = 170, 72, 104, 3
    adapters = {s: adapter(rng, rows, width, 16, True) for s in range(slots)}
    ids = np.sort(rng.integers(-1, slots, tokens)).astype(np.int32)
    x, base = inputs(rng, tokens, rows, width, True, "bf16")
    with AdapterBank(gpu_ctx, rows, width, slots, 16, tokens) as bank, ExpertDispatch(gpu_ctx, slots, 1, tokens) as d:
        fill(bank, rng, adapters)
        xd, idd, bd, yd = (gpu_ctx.upload(a) for a in (x, ids, base, np.full((tokens, rows), 0x1234, np.uint16)))
        d.plan_device(idd, tokens)
        gpu_ctx.copy_h2d(d.first, np.array(first, np.int32))
        bank.apply_device(xd, idd, tokens, bd, yd, plan=d.plan)
        assert (yd.download() == 0x1234).all()
        d.plan_device(idd, tokens)
        bank.apply_device(xd, idd, tokens, bd, yd, plan=d.plan)
        check(yd.download(), x, ids, base, adapters, True)
        for a in (xd, idd, bd, yd):
            a.free()


@pytest.mark.parametrize("max_rank", [32, 256])
def test_two_banks_on_two_streams_by_one_plan(gpu_ctx, max_rank):
    """A step's projections side by side: a bank and a stream each, the plan of the step's ids for both; adapters of the
    banks' largest rank and of small ones."""
    rng = np.random.default_rng(5)
    tokens, width, slots = 700, 264, 5
    ids = rng.integers(-1, slots, tokens).astype(np.int32)
    streams = [gpu_ctx.stream() for _ in range(2)]
    with ExpertDispatch(gpu_ctx, slots, 1, tokens) as d:
        idd, sides = gpu_ctx.upload(ids), []
        d.plan_device(idd, tokens)
        for rows, on in zip((200, 1032), streams):
            bank = AdapterBank(gpu_ctx, rows, width, slots, max_rank, tokens)
            adapters = {s: adapter(rng, rows, width, max_rank >> s, True) for s in range(slots)}
            fill(bank, rng, adapters)
            x, base = inputs(rng, tokens, rows, width, True, "f32")
            dev = [gpu_ctx.upload(a) for a in (x, base, np.zeros((tokens, rows), np.uint16))]
            sides.append((bank, adapters, x, base, dev, on))
        gpu_ctx.sync()
        for _ in range(5):
            for bank, _, _, _, (xd, bd, yd), on in sides:
                bank.apply_device(xd, idd, tokens, bd, yd, "f32", plan=d.plan, stream=on)
        gpu_ctx.sync()
        for bank, adapters, x, base, dev, on in sides:
            check(dev[2].download(), x, ids, base, adapters, True)
            for a in dev:
                a.free()
            bank.close()
            gpu_ctx.destroy_stream(on)
        idd.free()


@pytest.mark.parametrize("max_rank,dtype", [(4, "bf16"), (24, "f32"), (50, "bf16"), (100, "f32"), (200, "bf16")])
def test_most_slots(gpu_ctx, max_rank, dtype):
    """1024 slots. Many groups of two tokens, which make more tiles than the tokens would full ones; and all tokens of
    the last slot and one other, where nearly all groups that there could be make none."""
    rng = np.random.default_rng(max_rank)
    rows, width, slots = 8200, 72, 1024
    with AdapterBank(gpu_ctx, rows, width, slots, max_rank, 2100) as bank:
        adapters = {s: adapter(rng, rows, width, max_rank, True) for s in (*range(0, slots, 93), slots - 1)}
        fill(bank, rng, adapters)
        for tokens in (20, 2100):
            x, base = inputs(rng, tokens, rows, width, True, dtype)
            many = (np.arange(tokens) % slots).astype(np.int32)
            many[::3] = slots - 1
            for ids in (many, np.where(np.arange(tokens) % 5, slots - 1, 93).astype(np.int32)):
                check(bank.apply(x, ids, base), x, ids, base, adapters, True)


def test_call_refusals(gpu_ctx):
    rows, width, tokens = 64, 32, 4
    with AdapterBank(gpu_ctx, rows, width, 2, 8, tokens) as bank:
        a = 1 << 20   # addresses that no check follows
        good = dict(x=a, x_stride=width, ids=a, plan=None, tokens=tokens, base=2 * a, base_type=0, base_stride=rows,
                    y=3 * a, y_stride=rows, workspace=bank.workspace, workspace_bytes=bank.workspace_bytes)
        plan = _lib.MxRowPlan
        for changed in ({"x": None}, {"ids": None}, {"base": None}, {"y": None}, {"workspace": None}, {"tokens": -1},
                        {"tokens": (1 << 18) + 1}, {"base_type": 2}, {"x_stride": width - 8}, {"x_stride": width + 4},
                        {"base_stride": rows - 8}, {"base_stride": rows + 4}, {"base_type": 1, "base_stride": rows + 2},
                        {"y_stride": rows + 4}, {"y_stride": 8}, {"x": a + 8}, {"base": a + 8}, {"y": a + 2},
                        {"ids": a + 2}, {"workspace": bank.workspace + 16}, {"workspace_bytes": bank.workspace_bytes - 1},
                        {"y": a}, {"y": 2 * a, "y_stride": rows + 8}, {"y": 2 * a, "base_type": 1}, {"x_stride": 1 << 32},
                        {"plan": C.byref(plan(None, a, a))}, {"plan": C.byref(plan(a, a, None))},
                        {"plan": C.byref(plan(a + 2, a, a))}):
            args = dict(good, **changed)
            assert gpu_ctx.lib.cdll.mx_adapters_apply(bank.handle, *args.values(), None) == _lib.MX_ERR_INVALID, changed
        with pytest.raises(ValueError):   # a stride of zero is no default
            bank.apply_device(a, a, tokens, 2 * a, 3 * a, x_stride=0)
        for args in ((2, a, a, 8), (-1, a, a, 8), (0, a, a, 9), (0, a, a, -1), (0, None, a, 8), (0, a, None, 8),
                     (0, a + 1, a, 8)):
            assert gpu_ctx.lib.cdll.mx_adapters_load(bank.handle, *args, 1.0, None) == _lib.MX_ERR_INVALID, args
        for count in (0, -1, (1 << 18) + 1):
            assert gpu_ctx.lib.cdll.mx_adapters_workspace_bytes(bank.handle, count) == 0


def test_workspace_grows_with_the_tokens(gpu_ctx):
    """A bank sized for the most tokens holds every smaller call."""
    with AdapterBank(gpu_ctx, 64, 16384, 1, 256, 1) as bank:
        sizes = [bank.ctx.lib.cdll.mx_adapters_workspace_bytes(bank.handle, t) for t in range(1, 3000)]
    assert sizes == sorted(sizes)


def test_bank_memory_counts_and_goes_back():
    with _lib.Context(0, 64 << 20) as ctx:
        live = ctx.owned_bytes()[0]
        with AdapterBank(ctx, 512, 512, 4, 64, 8):
            assert ctx.owned_bytes()[0] >= live + 4 * 2 * 64 * 1024 * 2 // 2
        assert ctx.owned_bytes()[0] == live
        with pytest.raises(MemoryError):
            AdapterBank(ctx, 8192, 8192, 64, 256, 8)
        assert ctx.owned_bytes()[0] == live


@pytest.mark.parametrize("block", [32, 128])
def test_adapters_beside_fp8_projections(block):
    """fp8(name, values, adapters): the projection's own sums stay, and the output is those sums plus each row's adapter,
    rounded once; rows without one are the plain call's. The device form adds to the BF16 output in place."""
    rng = np.random.default_rng(block)
    layout = {"q_a": (192, 256), "o": (128, 384)}
    with NativeProjections(arrays_for(layout, block, rng), block=block, layout=layout) as proj:
        with pytest.raises(ValueError):
            proj.fp8("q_a", np.zeros((2, 256), np.uint16), np.zeros(2, np.int32))   # no bank yet
        for name, (rows, width) in layout.items():
            bank = proj.open_adapters(name, 3, 12, 160)
            with pytest.raises(RuntimeError):
                proj.open_adapters(name, 3, 12)
            adapters = {s: adapter(rng, rows, width, 4 * (s + 1), False) for s in range(2)}
            fill(bank, rng, adapters)
            for tokens in (1, 5, 50, 150):
                x = bf16_bits(rng.standard_normal((tokens, width)).astype(np.float32))
                ids = rng.integers(-1, 3, tokens).astype(np.int32)
                plain, got = proj.fp8(name, x), proj.fp8(name, x, ids)
                for stage in set(plain) - {"output_bf16"}:
                    np.testing.assert_array_equal(got[stage], plain[stage], err_msg=stage)
                check(got["output_bf16"], x, ids, plain["output_fp32"], adapters, False)
                without = ~np.isin(ids, list(adapters))
                np.testing.assert_array_equal(got["output_bf16"][without], plain["output_bf16"][without])
                dev = [proj.ctx.upload(a) for a in (x, ids, np.zeros((tokens, rows), np.uint16))]
                proj.project_device(name, dev[0], tokens, dev[2], adapters_ptr=dev[1])
                check(dev[2].download(), x, ids, plain["output_bf16"], adapters, False)
                for a in dev:
                    a.free()
            for bad in (np.zeros(3, np.int32), np.full(2, 3), np.zeros(2, np.float32)):
                with pytest.raises(ValueError):
                    proj.fp8(name, np.zeros((2, width), np.uint16), bad)
            with pytest.raises(ValueError):
                proj.fp8(name, np.zeros((161, width), np.uint16), np.zeros(161, np.int32))
            batched = proj.fp8(name, x.reshape(5, 30, width), ids.reshape(5, 30))["output_bf16"]
            np.testing.assert_array_equal(batched.reshape(150, rows), got["output_bf16"])
        proj.banks["o"].close()
        proj.open_adapters("o", 1, 4, 8)
    assert not proj.banks and proj.ctx is None
