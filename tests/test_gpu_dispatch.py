"""Tokens by expert and back on the device against the 64-bit oracle.

The plan and the moved rows are exact. A sum of n terms in FP32 is within n 2^-24 of the sum of the terms' magnitudes
(one rounding per addition, each at most half a step of a partial sum that the magnitudes bound; one more for a weighted
term's product); a BF16 result adds half a BF16 step, 2^-8 of its value. A weight's gradient is a dot product over the
row: in n = ceil(units / 1024) rounds of four units of up to eight values, a thread adds at most 32 n <= width / 256 + 32
products in order (units of one value: 4 n), six lane steps and up to three more waves follow, and each product was
rounded once.
"""

import ctypes as C

import numpy as np
import pytest

from oracle import dispatch as oracle
from oracle.formats import bf16_bits, bf16_values
from oracle.inputs import activations, mxfp4_expert
from tests.test_gpu_scratch import Graph
from vesper_amd import _lib
from vesper_amd.config import MoEConfig
from vesper_amd.dispatch import ExpertDispatch
from vesper_amd.layer import ExpertBank, MoELayer
from vesper_amd.moe import MoEAccumulator

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"bf16": 2.0 ** -8, "f32": 0.0}   # FP32 results are the FP32 sums themselves


def values(a):
    return bf16_values(a) if a.dtype == np.uint16 else a


def make_rows(rng, rows, width, dtype):
    if dtype == "u8":
        return rng.integers(0, 256, (rows, width)).astype(np.uint8)
    v = rng.standard_normal((rows, width)).astype(np.float32)
    return bf16_bits(v) if dtype == "bf16" else v


def routing(rng, tokens, k, experts, absent=True):
    """Ids with experts of other devices (negative and past the last) and repeated ones."""
    lo, hi = (-2, experts + 2) if absent else (0, experts)
    return rng.integers(lo, hi, (tokens, k)).astype(np.int32)


def check(got, want, size, terms, dtype):
    got = values(got).astype(np.float64)
    limit = np.abs(want) * HALF[dtype] + (1 + HALF[dtype]) * terms * U * size
    worst = np.max(np.abs(got - want) - limit) if got.size else 0.0
    assert worst <= 0, f"{worst:.3e} past the limit"


# (tokens, k, experts, width): one token, one pair, ragged counts and widths, more pairs than one walk of a wave, of a
# workgroup, and around powers of two; widths of whole 16-byte units and of single values
SHAPES = [(1, 1, 1, 1), (1, 8, 256, 7168), (2, 3, 5, 7), (7, 6, 384, 5120), (16, 8, 256, 136), (33, 32, 40, 24),
          (64, 2, 1024, 40), (127, 8, 16, 33), (129, 8, 256, 264), (255, 8, 3, 16), (300, 7, 100, 1000),
          (512, 4, 9, 8), (1025, 1, 17, 520), (2100, 8, 64, 12)]


@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32", "u8"])
def test_dispatch(gpu_ctx, tokens, k, experts, width, dtype):
    rng = np.random.default_rng(tokens * 31 + k)
    ids = routing(rng, tokens, k, experts)
    x = make_rows(rng, tokens, width, dtype)
    weights = rng.standard_normal((tokens, k)).astype(np.float32)
    with ExpertDispatch(gpu_ctx, experts, k, tokens) as d:
        got = d.dispatch(ids, x, weights)
    first, pair_row, row_pair = oracle.plan(ids, experts)
    np.testing.assert_array_equal(got["first"], first)
    np.testing.assert_array_equal(got["pair_row"], pair_row)
    np.testing.assert_array_equal(got["row_pair"], row_pair)
    n = first[-1]
    np.testing.assert_array_equal(got["rows"][:n], x[row_pair[:n] // k])
    np.testing.assert_array_equal(got["row_weights"][:n].view(np.uint32),
                                  weights.reshape(-1)[row_pair[:n]].view(np.uint32))
    assert not got["rows"][n:].any() and not got["row_weights"][n:].any()   # left as they were


@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("weighted,shared", [(False, False), (False, True), (True, False), (True, True)])
def test_combine(gpu_ctx, tokens, k, experts, width, dtype, weighted, shared):
    rng = np.random.default_rng(tokens * 17 + k)
    ids = routing(rng, tokens, k, experts)
    rows = make_rows(rng, tokens * k, width, dtype)
    weights = rng.standard_normal((tokens, k)).astype(np.float32) if weighted else None
    extra = make_rows(rng, tokens, width, dtype) if shared else None
    first, pair_row, _ = oracle.plan(ids, experts)
    rows[first[-1]:] = 0x7FC0 if dtype == "bf16" else np.nan   # rows that no token has are not read
    with ExpertDispatch(gpu_ctx, experts, k, tokens) as d:
        d.dispatch(ids, np.zeros((tokens, 1), np.uint8))
        got = d.combine(rows, weights, extra)
    want, size = oracle.combine(values(rows), pair_row, weights, None if extra is None else values(extra))
    check(got, want, size, k + 2, dtype)


@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("weighted", [False, True])
def test_combine_backward(gpu_ctx, tokens, k, experts, width, dtype, weighted):
    rng = np.random.default_rng(tokens * 13 + k)
    ids = routing(rng, tokens, k, experts)
    rows, dy = make_rows(rng, tokens * k, width, dtype), make_rows(rng, tokens, width, dtype)
    weights = rng.standard_normal((tokens, k)).astype(np.float32) if weighted else None
    with ExpertDispatch(gpu_ctx, experts, k, tokens) as d:
        d.dispatch(ids, np.zeros((tokens, 1), np.uint8))
        got = d.combine_backward(dy, rows, weights)
    first, pair_row, _ = oracle.plan(ids, experts)
    drows, dweights, size = oracle.combine_backward(values(dy), values(rows), pair_row, weights)
    check(got["drows"], drows, np.abs(drows), 1, dtype)
    assert not got["drows"][first[-1]:].any()
    depth = -(-width // 256) + 32 + 6 + 3
    check(got["dweights"], dweights, size, depth + 1, "f32")


@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_dispatch_backward(gpu_ctx, tokens, k, experts, width, dtype):
    rng = np.random.default_rng(tokens * 11 + k)
    ids = routing(rng, tokens, k, experts)
    drows = make_rows(rng, tokens * k, width, dtype)
    drow_weights = rng.standard_normal(tokens * k).astype(np.float32)
    with ExpertDispatch(gpu_ctx, experts, k, tokens) as d:
        d.dispatch(ids, np.zeros((tokens, 1), np.uint8))
        got = d.dispatch_backward(drows, drow_weights)
    _, pair_row, _ = oracle.plan(ids, experts)
    want, size = oracle.combine(values(drows), pair_row)
    check(got["dx"], want, size, k, dtype)
    picked = np.where(pair_row >= 0, drow_weights[np.maximum(pair_row, 0)], np.float32(0))
    np.testing.assert_array_equal(got["dweights"], picked)


def test_gradients_against_differences(gpu_ctx):
    """The loss <combine(rows, w), dy> is linear in each entry, so a step of 1 gives its gradient up to the FP32 sums'
    rounding on either side."""
    rng = np.random.default_rng(5)
    ids = np.array([[1, 0], [2, 9], [0, 0]], np.int32)
    rows, dy = make_rows(rng, 6, 8, "f32"), make_rows(rng, 3, 8, "f32")
    weights = rng.standard_normal((3, 2)).astype(np.float32)
    with ExpertDispatch(gpu_ctx, 3, 2, 3) as d:
        d.dispatch(ids, np.zeros((3, 1), np.uint8))
        got = d.combine_backward(dy, rows, weights)
        loss = lambda r, w: (d.combine(r, w).astype(np.float64) * dy).sum()  # noqa: E731
        # a term is at most (|row| + 1)(|w| + 1), 3 terms a sum, 24 sums: rounding below 24 * 4 * 2^-24 * 40
        limit = 2 * 24 * 4 * U * 40
        for r in range(6):
            step = np.zeros_like(rows)
            step[r, r] = 1
            assert abs(loss(rows + step, weights) - loss(rows, weights) - got["drows"][r, r]) < limit
        for index in np.ndindex(3, 2):
            step = np.zeros_like(weights)
            step[index] = 1
            assert abs(loss(rows, weights + step) - loss(rows, weights) - got["dweights"][index]) < limit


# pairs around the sizes where another form of the plan takes over (8192, 16384, 49152 over the rounds of 512 groups), and
# routings that put all pairs in one group or in none
@pytest.mark.parametrize("tokens,k,experts", [(1025, 8, 30), (2049, 8, 30), (6143, 8, 256), (6145, 8, 256), (49153, 1, 17),
                                              (70001, 1, 1), (1537, 16, 512), (2051, 8, 1024), (40000, 32, 1023)])
@pytest.mark.parametrize("kind", ["random", "one", "none"])
def test_plans_of_many_pairs(gpu_ctx, tokens, k, experts, kind):
    rng = np.random.default_rng(tokens)
    ids = routing(rng, tokens, k, experts)
    if kind != "random":
        ids[:] = experts - 1 if kind == "one" else experts
        ids[tokens // 2] = 0
    key = np.where((ids >= 0) & (ids < experts), ids, experts).reshape(-1)
    row_pair = np.argsort(key, kind="stable")
    first = np.searchsorted(key[row_pair], np.arange(experts + 1))
    pair_row = np.full(tokens * k, -1)
    pair_row[row_pair[:first[-1]]] = np.arange(first[-1])
    idd = gpu_ctx.upload(ids)
    with ExpertDispatch(gpu_ctx, experts, k, tokens) as d:
        for _ in range(2):   # the second over the first's plan
            d.plan_device(idd, tokens)
        got = d.read_plan()
    idd.free()
    for name, want in (("first", first), ("pair_row", pair_row.reshape(tokens, k)), ("row_pair", row_pair)):
        np.testing.assert_array_equal(got[name], want)


def test_no_token_and_no_row(gpu_ctx):
    with ExpertDispatch(gpu_ctx, 6, 2, 8) as d:
        got = d.dispatch(np.zeros((0, 2), np.int32), np.zeros((0, 64), np.uint16))
        np.testing.assert_array_equal(got["first"], np.zeros(7))
        assert d.combine(np.zeros((0, 64), np.uint16)).shape == (0, 64)
        # every pair belongs elsewhere: nothing moves, the sums are zero (the shared row alone), gradients zero
        x = make_rows(np.random.default_rng(0), 5, 64, "bf16")
        got = d.dispatch(np.full((5, 2), -1, np.int32), x)
        assert got["first"][-1] == 0 and not got["rows"].any()
        nan = np.full((10, 64), 0x7FC0, np.uint16)
        assert not d.combine(nan).any()
        np.testing.assert_array_equal(d.combine(nan, None, x), x)
        back = d.combine_backward(x, nan, np.ones((5, 2)))
        assert not back["drows"].any() and not back["dweights"].any()
        assert not d.dispatch_backward(nan)["dx"].any()


def test_nan_and_infinity_stay_in_their_row(gpu_ctx):
    rows = np.ones((4, 8), np.float32)
    rows[1, 2], rows[2, 3] = np.nan, -np.inf
    ids = np.array([[0, 1], [1, 0]], np.int32)   # rows 0, 1: expert 0 of tokens 0, 1; rows 2, 3: expert 1
    with ExpertDispatch(gpu_ctx, 2, 2, 2) as d:
        d.dispatch(ids, np.zeros((2, 1), np.uint8))
        y = d.combine(rows)
    assert np.isnan(y[1, 2]) and np.isneginf(y[0, 3])
    y[1, 2] = y[0, 3] = 2
    np.testing.assert_array_equal(y, np.full((2, 8), 2, np.float32))


@pytest.mark.parametrize("dtype,offset,width", [("bf16", 1, 64), ("bf16", 2, 64), ("f32", 1, 32), ("u8", 3, 160),
                                                ("bf16", 8, 64)])
def test_rows_at_any_element(gpu_ctx, dtype, offset, width):
    """Buffers that start `offset` elements into an allocation, surrounded by values that have to stay."""
    rng = np.random.default_rng(offset)
    t, k, e = 9, 3, 5
    x = make_rows(rng, t, width, dtype)
    size = x.dtype.itemsize
    ids = routing(rng, t, k, e)
    first, pair_row, row_pair = oracle.plan(ids, e)
    n = first[-1]
    flat = lambda a, rows: np.concatenate([np.full(offset, 77, a.dtype), a.ravel(), np.full(99, 77, a.dtype)])[  # noqa: E731
        :offset + rows * width + 99]
    xd, rd = gpu_ctx.upload(flat(x, t)), gpu_ctx.upload(flat(np.full((t * k, width), 77, x.dtype), t * k))
    idd = gpu_ctx.upload(ids)
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        d.dispatch_device(idd, t, xd.ptr + offset * size, width, rd.ptr + offset * size, dtype)
        got = rd.download()
        np.testing.assert_array_equal(got[:offset], np.full(offset, 77, x.dtype))
        body = got[offset:offset + t * k * width].reshape(t * k, width)
        np.testing.assert_array_equal(body[:n], x[row_pair[:n] // k])
        assert (body[n:] == 77).all() and (got[offset + t * k * width:] == 77).all()
        if dtype != "u8":
            d.combine_device(rd.ptr + offset * size, width, xd.ptr + offset * size, dtype)
            y = xd.download()
            want, total = oracle.combine(values(body), pair_row)
            check(y[offset:offset + t * width].reshape(t, width), want, total, k, dtype)
            assert (y[:offset] == 77).all() and (y[offset + t * width:] == 77).all()
    for a in (xd, rd, idd):
        a.free()


def test_in_place_forms(gpu_ctx):
    """y may be the shared rows, drows the rows: the same results as apart."""
    rng = np.random.default_rng(8)
    t, k, e, width = 21, 4, 6, 264
    ids = routing(rng, t, k, e)
    rows, dy, shared = (make_rows(rng, n, width, "bf16") for n in (t * k, t, t))
    weights = rng.standard_normal((t, k)).astype(np.float32)
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        n = d.dispatch(ids, dy)["first"][-1]
        y, back = d.combine(rows, weights, shared), d.combine_backward(dy, rows, weights)
        dev = [gpu_ctx.upload(a) for a in (rows, dy, shared, weights, np.zeros((t, k), np.float32))]
        rd, gd, sd, wd, dwd = dev
        d.combine_device(rd, width, sd, "bf16", wd, sd)
        np.testing.assert_array_equal(sd.download(), y)
        d.combine_backward_device(gd, rd, width, rd, dwd, "bf16", wd)
        np.testing.assert_array_equal(rd.download()[:n], back["drows"][:n])
        np.testing.assert_array_equal(dwd.download().view(np.uint32), back["dweights"].view(np.uint32))
        # either gradient alone
        d.combine_backward_device(gd, None, width, rd, None, "bf16", wd)
        np.testing.assert_array_equal(rd.download()[:n], back["drows"][:n])
        rd.upload(rows)
        d.combine_backward_device(gd, rd, width, None, dwd, "bf16", wd)
        np.testing.assert_array_equal(dwd.download().view(np.uint32), back["dweights"].view(np.uint32))
        np.testing.assert_array_equal(rd.download(), rows)
        for a in dev:
            a.free()


def test_codes_and_scales_move_by_one_plan(gpu_ctx):
    rng = np.random.default_rng(9)
    t, k, e = 40, 6, 12
    ids = routing(rng, t, k, e)
    codes, scales = make_rows(rng, t, 5120, "u8"), make_rows(rng, t, 160, "u8")
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        got = d.dispatch(ids, codes)
        n, token = got["first"][-1], got["row_pair"] // k
        sd, rd = gpu_ctx.upload(scales), gpu_ctx.upload(np.zeros((t * k, 160), np.uint8))
        d.move_device(sd, 160, rd, "u8")
        np.testing.assert_array_equal(rd.download()[:n], scales[token[:n]])
        np.testing.assert_array_equal(got["rows"][:n], codes[token[:n]])
        sd.free()
        rd.free()


def test_a_plan_with_rows_out_of_range_reads_and_writes_nothing_there(gpu_ctx):
    """pair_row is device memory a caller may have spoiled: rows outside [0, T k) count as absent."""
    t, k, width = 3, 2, 64
    spoiled = np.array([[0, 6], [-7, 1], [2 ** 30, 2]], np.int32)
    rows = make_rows(np.random.default_rng(1), t * k, width, "f32")
    with ExpertDispatch(gpu_ctx, 4, k, t) as d:
        d.dispatch(np.zeros((t, k), np.int32), np.zeros((t, 1), np.uint8))
        gpu_ctx.copy_h2d(d.pair_row, spoiled)
        kept = np.where((spoiled >= 0) & (spoiled < t * k), spoiled, -1)
        np.testing.assert_array_equal(d.combine(rows), oracle.combine(rows, kept)[0].astype(np.float32))
        back = d.combine_backward(np.ones((t, width), np.float32), rows)
        assert (back["drows"][[0, 1, 2]] == 1).all() and not back["drows"][3:].any()
        assert (back["dweights"][kept < 0] == 0).all()


def test_combine_is_the_accumulator(gpu_ctx):
    """Without weights: MoEAccumulator's sums, bit for bit."""
    rng = np.random.default_rng(12)
    t, k, e, width = 11, 6, 24, 256
    ids = np.stack([rng.permutation(e)[:k] for _ in range(t)]).astype(np.int32)
    rows, shared = make_rows(rng, t * k, width, "bf16"), make_rows(rng, t, width, "bf16")
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        plan = d.dispatch(ids, shared)
        got = d.combine(rows, None, shared)
    first = plan["first"]
    with MoEAccumulator(hidden=width, experts=e, top_k=k) as acc:
        parts = {i: rows[first[i]:first[i + 1]] for i in range(e) if first[i] < first[i + 1]}
        np.testing.assert_array_equal(got, acc.run(ids, parts, shared)["output_bf16"])


def test_experts_between_dispatch_and_combine_are_the_layer(gpu_ctx):
    """Route, dispatch with the route weights, every expert on its slice of the rows, combine with the shared expert:
    the routed decode layer's output on the same weights, bit for bit (its expert rows do not depend on the batch)."""
    rng = np.random.default_rng(21)
    cfg = MoEConfig(hidden=512, intermediate=256, experts=12, top_k=4, max_tokens=13)
    t, h = 13, cfg.hidden
    x = bf16_bits(activations(rng, t, h))
    ids = np.stack([rng.permutation(cfg.experts)[:cfg.top_k] for _ in range(t)]).astype(np.int32)
    weights = rng.uniform(0.1, 1.0, ids.shape).astype(np.float32)
    bank = ExpertBank(gpu_ctx, cfg, cfg.experts + 1)
    for e in range(cfg.experts + 1):
        bank.upload(e, mxfp4_expert(rng, h, cfg.intermediate))
    lib, ctx = gpu_ctx.lib, gpu_ctx._h()
    dev = {n: gpu_ctx.upload(a) for n, a in (
        ("x", x), ("ids", ids), ("w", weights), ("rows", np.zeros((t * cfg.top_k, h), np.uint16)),
        ("rw", np.zeros(t * cfg.top_k, np.float32)), ("out", np.zeros((t * cfg.top_k, h), np.uint16)),
        ("shared", np.zeros((t, h), np.uint16)), ("y", np.zeros((t, h), np.uint16)))}

    def expert(e, at, rows, route, to):
        lib.expert_forward_tiled(ctx, C.c_void_p(bank.tiled_ptr(e)), h, cfg.intermediate, C.c_void_p(at), rows,
                                 cfg.swiglu_limit, route, C.c_void_p(to), None, None)

    with ExpertDispatch(gpu_ctx, cfg.experts, cfg.top_k, t) as d, \
            MoELayer(gpu_ctx, cfg, np.zeros((cfg.experts, h), np.float32), bank) as layer:
        d.dispatch_device(dev["ids"], t, dev["x"], h, dev["rows"], "bf16", dev["w"], dev["rw"])
        first = d.read_plan()["first"]
        for e in range(cfg.experts):
            if first[e] < first[e + 1]:
                at = int(first[e])
                expert(e, dev["rows"].ptr + 2 * h * at, int(first[e + 1]) - at, C.c_void_p(dev["rw"].ptr + 4 * at),
                       dev["out"].ptr + 2 * h * at)
        expert(cfg.experts, dev["x"].ptr, t, None, dev["shared"].ptr)
        d.combine_device(dev["out"], h, dev["y"], "bf16", None, dev["shared"])
        got = dev["y"].download()
        lib.moe_decode_routed(layer.handle, _lib.vp(dev["x"]), t, _lib.vp(dev["ids"]), _lib.vp(dev["w"]),
                              _lib.vp(dev["y"]), None)
        np.testing.assert_array_equal(got, dev["y"].download())
        assert got.any() and layer.route_errors() == 0
    for a in dev.values():
        a.free()
    bank.free()


@pytest.mark.parametrize("tokens", [3, 400, 7000])
def test_captured_passes_replay_on_new_inputs(gpu_ctx, tokens):
    """Forward and backward captured once on a stream of their own; each replay reads what the buffers then hold."""
    k, e, width = 8, 20, 136
    with _lib.Context(0) as ctx:
        stream = ctx.stream()
        shapes = {"ids": ((tokens, k), np.int32), "x": ((tokens, width), np.float32), "w": ((tokens, k), np.float32),
                  "rows": ((tokens * k, width), np.float32), "rw": ((tokens * k,), np.float32),
                  "y": ((tokens, width), np.float32), "drows": ((tokens * k, width), np.float32),
                  "dw": ((tokens, k), np.float32), "dx": ((tokens, width), np.float32)}
        dev = {n: ctx.upload(np.zeros(*s)) for n, s in shapes.items()}
        with ExpertDispatch(ctx, e, k, tokens) as d:
            def passes(on):
                d.dispatch_device(dev["ids"], tokens, dev["x"], width, dev["rows"], "f32", dev["w"], dev["rw"],
                                  stream=on)
                d.combine_device(dev["rows"], width, dev["y"], "f32", dev["w"], stream=on)
                d.combine_backward_device(dev["y"], dev["rows"], width, dev["drows"], dev["dw"], "f32", dev["w"],
                                          stream=on)
                d.dispatch_backward_device(dev["drows"], width, dev["dx"], "f32", stream=on)

            graph = Graph(ctx, stream, lambda: passes(stream))
            for replay in range(4):
                rng = np.random.default_rng(replay)
                dev["ids"].upload(routing(rng, tokens, k, e))
                dev["x"].upload(make_rows(rng, tokens, width, "f32"))
                dev["w"].upload(rng.standard_normal((tokens, k)).astype(np.float32))
                ctx.sync()
                graph.launch()
                got = [dev[n].download() for n in ("y", "dw", "dx")]
                passes(None)
                for g, n in zip(got, ("y", "dw", "dx")):
                    np.testing.assert_array_equal(g, dev[n].download(), err_msg=n)
            graph.close()
        for a in dev.values():
            a.free()
        ctx.destroy_stream(stream)


def test_two_dispatches_on_two_streams(gpu_ctx):
    """Objects of their own, streams of their own: neither call's plan or rows reach the other."""
    rng = np.random.default_rng(3)
    t, k, e, width = 700, 4, 30, 128
    streams = [gpu_ctx.stream() for _ in range(2)]
    sides = []
    for on in streams:
        ids, x = routing(rng, t, k, e), make_rows(rng, t, width, "bf16")
        dev = [gpu_ctx.upload(a) for a in (ids, x, np.zeros((t * k, width), np.uint16), np.zeros((t, width), np.uint16))]
        sides.append((ids, x, dev, ExpertDispatch(gpu_ctx, e, k, t), on))
    gpu_ctx.sync()
    for _ in range(5):
        for _, _, (idd, xd, rd, yd), d, on in sides:
            d.dispatch_device(idd, t, xd, width, rd, stream=on)
            d.combine_device(rd, width, yd, stream=on)
    gpu_ctx.sync()
    for ids, x, dev, d, _ in sides:
        first, pair_row, row_pair = oracle.plan(ids, e)
        np.testing.assert_array_equal(dev[2].download()[:first[-1]], x[row_pair[:first[-1]] // k])
        want, size = oracle.combine(values(dev[2].download()), pair_row)
        check(dev[3].download(), want, size, k, "bf16")
        d.close()
        for a in dev:
            a.free()
    for on in streams:
        gpu_ctx.destroy_stream(on)


def test_rows_past_32_bits(gpu_ctx):
    """More than 2^31 values in the rows: the first and last tokens' are the ones looked at."""
    rng = np.random.default_rng(6)
    t, k, width = 600, 2, 1 << 21
    ids = np.stack([np.arange(t) % 7, 7 + np.arange(t) % 5], 1).astype(np.int32)   # two groups each, all held
    w = rng.uniform(0.5, 1, (t, k)).astype(np.float32)
    looked = (0, 1, t // 2, t - 2, t - 1)
    xs = {i: make_rows(rng, 1, width, "bf16")[0] for i in looked}
    first, pair_row, row_pair = oracle.plan(ids, 12)
    assert int(pair_row.max()) * width > 1 << 31
    with ExpertDispatch(gpu_ctx, 12, k, t) as d:
        row = 2 * width
        xd, yd, rd = gpu_ctx.malloc(t * row), gpu_ctx.malloc(t * row), gpu_ctx.malloc(t * k * row)
        idd, wd, dwd = gpu_ctx.upload(ids), gpu_ctx.upload(w), gpu_ctx.upload(np.zeros((t, k), np.float32))
        for i, x in xs.items():
            gpu_ctx.copy_h2d(xd + i * row, x)
        d.dispatch_device(idd, t, xd, width, rd)
        for i, x in xs.items():
            for j in range(k):
                np.testing.assert_array_equal(gpu_ctx.download(rd + int(pair_row[i, j]) * row, (width,), np.uint16), x)
        d.combine_device(rd, width, yd, weights_ptr=wd)
        for i, x in xs.items():
            want = np.stack([np.float64(w[i, j]) * values(x) for j in range(k)])
            check(gpu_ctx.download(yd + i * row, (width,), np.uint16), want.sum(0), np.abs(want).sum(0), k + 1, "bf16")
        d.combine_backward_device(xd, rd, width, rd, dwd, weights_ptr=wd)
        dw = dwd.download()
        for i, x in xs.items():
            v = values(x).astype(np.float64)
            for j in range(k):
                got = gpu_ctx.download(rd + int(pair_row[i, j]) * row, (width,), np.uint16)
                check(got, w[i, j] * v, np.abs(w[i, j] * v), 1, "bf16")
                assert abs(dw[i, j] - v @ v) <= (width / 256 + 32 + 10) * U * (v @ v)
        d.dispatch_backward_device(rd, width, yd)
        for i in xs:
            terms = [values(gpu_ctx.download(rd + int(r) * row, (width,), np.uint16)).astype(np.float64) for r in pair_row[i]]
            check(gpu_ctx.download(yd + i * row, (width,), np.uint16), sum(terms), sum(map(np.abs, terms)), k, "bf16")
        for a in (idd, wd, dwd):
            a.free()
        for p in (xd, yd, rd):
            gpu_ctx.free(p)


def test_most_pairs(gpu_ctx):
    """The largest routing: 2^18 tokens of 32 of 1024 experts, rows of one byte."""
    rng = np.random.default_rng(7)
    t, k, e = 1 << 18, 32, 1024
    ids, x = routing(rng, t, k, e), make_rows(rng, t, 1, "u8")
    key = np.where((ids >= 0) & (ids < e), ids, e).reshape(-1)
    row_pair = np.argsort(key, kind="stable")
    first = np.searchsorted(key[row_pair], np.arange(e + 1))
    pair_row = np.full(t * k, -1)
    pair_row[row_pair[:first[e]]] = np.arange(first[e])
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        out = d.dispatch(ids, x)
    for name, want in (("first", first), ("pair_row", pair_row.reshape(t, k)), ("row_pair", row_pair)):
        np.testing.assert_array_equal(out[name], want)
    np.testing.assert_array_equal(out["rows"][:first[-1]], x[row_pair[:first[-1]] // k])


@pytest.mark.parametrize("dtype,width", [("bf16", 7168), ("f32", 3584), ("bf16", 7161)])
def test_calls_larger_than_the_caches(gpu_ctx, dtype, width):
    """Calls that move more than 96 MiB take their rows past the caches; tokens with all their pairs and without some."""
    rng = np.random.default_rng(width)
    t, k, e = 900, 8, 64
    ids = routing(rng, t, k, e, absent=False)
    ids[::5] = routing(rng, len(ids[::5]), k, e)
    x, w = make_rows(rng, t, width, dtype), rng.standard_normal((t, k)).astype(np.float32)
    with ExpertDispatch(gpu_ctx, e, k, t) as d:
        out = d.dispatch(ids, x)
        first, pair_row, row_pair = oracle.plan(ids, e)
        np.testing.assert_array_equal(out["rows"][:first[-1]], x[row_pair[:first[-1]] // k])
        rows = make_rows(rng, t * k, width, dtype)
        want, size = oracle.combine(values(rows), pair_row, w, values(x))
        check(d.combine(rows, w, x), want, size, k + 2, dtype)
        got = d.combine_backward(x, rows, w)
        v, held = values(x).astype(np.float64), pair_row >= 0
        want = w.reshape(-1, 1)[row_pair[:first[-1]]] * v[row_pair[:first[-1]] // k]
        check(got["drows"][:first[-1]], want, np.abs(want), 1, dtype)
        r = values(rows).astype(np.float64)[np.where(held, pair_row, 0)]   # [T, k, width]
        dot, size = np.einsum("tjw,tw->tj", r, v), np.einsum("tjw,tw->tj", np.abs(r), np.abs(v))
        assert np.all(np.abs(got["dweights"] - np.where(held, dot, 0)) <= np.where(held, (width / 256 + 42) * U * size, 0))
        want, size = oracle.combine(values(rows), pair_row)
        check(d.dispatch_backward(rows)["dx"], want, size, k, dtype)
