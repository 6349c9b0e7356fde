"""Heads normalized and rotated, and their gradients, on the device against the 64-bit oracle.

Every value passes at most 8 FP32 roundings after the root (its own, three products, two products and a sum of the turn):
8 2^-24 of |a| + |b|, the pair's normalized magnitudes; a BF16 result is half a step, 2^-8 of its value, from there. A
gradient's mean is a chain of at most width / L + log2 L <= 80 additions of products that have two roundings each; dweight is
a chain of at most rows / 512 + 4 + 32 + 48 additions (a lane's rows, the workgroup's groups, the workgroups' parts).
"""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_values
from tests.test_gpu_scratch import Graph
from vesper_amd import _lib
from vesper_amd.attention import HeadRotation, rotation_table

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def values(a):
    return bf16_values(a).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


def typed(a, dtype):
    return bf16_bits(a.astype(np.float32)) if dtype == "bf16" else a.astype(np.float32)


def magnitude(x, first, dims, style):
    """|a| + |b| of each rotated value's pair, |x| elsewhere."""
    m = np.abs(np.array(x, np.float64))
    i = np.arange(dims // 2)
    a, b = (first + i, first + i + dims // 2) if style == "halves" else (first + 2 * i, first + 2 * i + 1)
    both = m[..., a] + m[..., b]
    m[..., a] = m[..., b] = both
    return m


def within(got, want, limit, dtype):
    got, limit = values(got), limit + 1e-37
    if dtype == "bf16":
        limit = limit + 2.0 ** -8 * (np.abs(want) + limit)
    assert np.all(np.abs(got - want) <= limit), np.max(np.abs(got - want) - limit)


# (tokens, heads, width, norm, first, dims, style): each number of lanes and steps a row can take, norms and rotations of a
# part, next to or over each other, of nothing
CASES = [(1, 1, 8, 8, 0, 8, "pairs"), (1, 64, 512, 512, 448, 64, "pairs"), (7, 3, 64, 64, 0, 64, "halves"), (5, 2, 48, 48, 16, 32, "halves"),
         (33, 5, 128, 128, 0, 128, "halves"), (100, 7, 192, 0, 128, 64, "pairs"), (19, 2, 576, 512, 512, 64, "pairs"),
         (3, 2, 576, 64, 32, 512, "halves"), (11, 1, 1024, 1024, 0, 0, "pairs"), (2, 3, 1280, 1280, 1264, 16, "halves"),
         (2, 1, 4096, 4096, 0, 4096, "halves"), (4, 2, 4096, 8, 4088, 8, "pairs"), (600, 40, 128, 128, 96, 32, "pairs"),
         (9, 4, 72, 40, 8, 64, "halves"), (2, 2, 256, 0, 0, 0, "pairs"), (1500, 3, 64, 64, 32, 32, "halves")]


def case_of(tokens, heads, width, norm, first, dims, style, dtype, seed=0):
    rng = np.random.default_rng(tokens * 7 + width + seed)
    x = values(typed(rng.standard_normal((tokens, heads, width)) * np.exp2(rng.integers(-6, 7, (tokens, heads, 1))), dtype))
    table = rotation_table(50, dims) if dims else None
    positions = rng.integers(0, 50, tokens)
    weight = rng.uniform(0.5, 1.5, norm).astype(np.float32) if norm else None
    return rng, x, table, positions, weight


@pytest.mark.parametrize("tokens,heads,width,norm,first,dims,style", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_apply(gpu_ctx, tokens, heads, width, norm, first, dims, style, dtype):
    rng, x, table, positions, weight = case_of(tokens, heads, width, norm, first, dims, style, dtype)
    with HeadRotation(gpu_ctx, width, norm, dims, first, style, table=table) as rot:
        for w, inverse in ((weight, False), (None, True)):
            got = rot.apply(typed(x, dtype), positions if dims else None, w, inverse)
            args = dict(norm=norm, weight=w, first=first, dims=dims, style=style)
            want = oracle.heads(x, table, positions, inverse=inverse, **args)
            size = magnitude(oracle.heads(x, norm=norm, weight=w), first, dims, style)
            within(got, want, 8 * U * size, dtype)


@pytest.mark.parametrize("tokens,heads,width,norm,first,dims,style", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward(gpu_ctx, tokens, heads, width, norm, first, dims, style, dtype):
    rng, x, table, positions, weight = case_of(tokens, heads, width, norm, first, dims, style, dtype, 1)
    dy = values(typed(rng.standard_normal(x.shape), dtype))
    with HeadRotation(gpu_ctx, width, norm, dims, first, style, table=table) as rot:
        for w, inverse in ((weight, False), (None, True)):
            got = rot.backward(typed(dy, dtype), typed(x, dtype), positions if dims else None, w, inverse)
            args = dict(norm=norm, weight=w, first=first, dims=dims, style=style)
            dx, dw = oracle.heads_backward(dy, x, table, positions, inverse=inverse, **args)
            size = magnitude(dy, first, dims, style)
            limit = 8 * U * size
            if norm:
                r = 1 / np.sqrt(np.mean(x[..., :norm] ** 2, -1, keepdims=True) + 1e-6)
                u, gw = np.abs(x[..., :norm] * r), size[..., :norm] * (1 if w is None else w)
                mean = np.mean(gw * u, -1, keepdims=True)
                limit[..., :norm] = r * U * (16 * gw + u * mean * (80 + 16))
                chain = tokens * heads / 512 + 84 + 16
                assert np.all(np.abs(got["dweight"] - dw) <= chain * U * np.sum(size[..., :norm] * u, (0, 1)) + 1e-37)
            within(got["dx"], dx, limit, dtype)


def test_root_of_tiny_and_huge_rows(gpu_ctx):
    """Means outside FP32's normal range, a row of zeros with no eps, and eps alone."""
    x = np.zeros((5, 1, 64), np.float32)
    x[0], x[1], x[2, 0, 3] = 1e-30, 1e30, 3e38
    x[3] = 1e-22
    with HeadRotation(gpu_ctx, 64, 64, eps=0.0) as rot:
        got = rot.apply(x)
    want = oracle.heads(x[:4], norm=64, eps=0.0)
    np.testing.assert_allclose(got[:4], want, rtol=8 * U)
    assert np.isnan(got[4]).all()
    with HeadRotation(gpu_ctx, 64, 64, eps=1e-6) as rot:
        np.testing.assert_allclose(rot.apply(x), oracle.heads(x, norm=64, eps=1e-6), rtol=8 * U, atol=1e-40)


def test_queries_and_keys_in_one_call_of_strided_rows_on_a_stream(gpu_ctx):
    """Column ranges of one projection output with weights of each, odd strides and offsets, captured and replayed; the
    gradients likewise."""
    rng, t, w = np.random.default_rng(5), 37, 128
    table = rotation_table(40, 64)
    positions = rng.integers(0, 40, t).astype(np.int32)
    weights = [rng.uniform(.5, 1.5, w).astype(np.float32) for _ in range(2)]
    for lead, dtype, stride in ((0, "f32", 11 * w), (3, "f32", 11 * w + 5), (0, "bf16", 11 * w + 8), (1, "bf16", 11 * w + 3)):
        size = 4 if dtype == "f32" else 2
        x = typed(rng.standard_normal((t, stride)), dtype)
        dy = typed(rng.standard_normal((t, stride)), dtype)
        spans = [(lead, 8), (lead + 8 * w, 3)]
        y0 = typed(np.full((t, stride), 7.0), dtype)
        with HeadRotation(gpu_ctx, w, w, 64, 0, "halves", table=table) as rot:
            dev = [gpu_ctx.upload(a) for a in (x, y0, positions, *weights, dy, y0, np.zeros((2, w), np.float32))]
            dx_, dy_ = dev[6], dev[5]
            rot.open_gradients()
            stream = gpu_ctx.stream()

            def call():
                sets = [rot.set(dev[0].ptr + at * size, h, dev[1].ptr + at * size, dev[3 + i], stride, stride)
                        for i, (at, h) in enumerate(spans)]
                rot.apply_device(sets, t, dev[2], dtype, stream=stream)
                grads = [rot.grad(dev[0].ptr + at * size, h, dy_.ptr + at * size, dx_.ptr + at * size, dev[3 + i],
                                  dev[7].ptr + 4 * w * i, stride, stride, stride) for i, (at, h) in enumerate(spans)]
                rot.backward_device(grads, t, dev[2], dtype, stream=stream)
            graph = Graph(gpu_ctx, stream, call)
            for replay in range(3):
                for d in (dev[1], dx_):
                    d.upload(y0)
                dev[7].upload(np.zeros((2, w), np.float32))
                gpu_ctx.sync()
                graph.launch()
                got, dgot, dwgot = dev[1].download(), dx_.download(), dev[7].download()
                touched = np.zeros(stride, bool)
                for i, (at, h) in enumerate(spans):
                    cols = slice(at, at + h * w)
                    touched[cols] = True
                    xi, gi = values(x[:, cols]).reshape(t, h, w), values(dy[:, cols]).reshape(t, h, w)
                    args = dict(norm=w, weight=weights[i], first=0, dims=64, style="halves")
                    want = oracle.heads(xi, table, positions, **args)
                    within(got[:, cols].reshape(t, h, w), want, 8 * U * magnitude(oracle.heads(xi, norm=w, weight=weights[i]), 0, 64, "halves"), dtype)
                    dx, dw = oracle.heads_backward(gi, xi, table, positions, **args)
                    r = 1 / np.sqrt(np.mean(xi ** 2, -1, keepdims=True) + 1e-6)
                    gw = magnitude(gi, 0, 64, "halves") * weights[i]
                    u = np.abs(xi * r)
                    within(dgot[:, cols].reshape(t, h, w), dx, r * U * (16 * gw + 96 * u * np.mean(gw * u, -1, keepdims=True)), dtype)
                    assert np.all(np.abs(dwgot[i] - dw) <= 100 * U * np.sum(gw / weights[i] * u, (0, 1)))
                for a in (got, dgot):
                    np.testing.assert_array_equal(a[:, ~touched], y0[:, ~touched])
            graph.close()
            gpu_ctx.destroy_stream(stream)
            for d in dev:
                d.free()


def test_rows_of_no_token(gpu_ctx):
    """Positions outside the table: y as it was, dx zero, nothing in dweight; for every row of a call as well."""
    rng, table = np.random.default_rng(6), rotation_table(8, 16)
    x, dy = rng.standard_normal((2, 6, 2, 64)).astype(np.float32)
    w = rng.uniform(.5, 1.5, 64).astype(np.float32)
    for positions in (np.array([0, 8, 3, -1, 7, 2 ** 31 - 1]), np.full(6, -2 ** 31)):
        live = (positions >= 0) & (positions < 8)
        with HeadRotation(gpu_ctx, 64, 64, 16, table=table) as rot:
            dev = [gpu_ctx.upload(a) for a in (x, np.full_like(x, 7), positions.astype(np.int32), w, dy, np.full_like(x, 7), np.full(64, 7, np.float32))]
            rot.apply_device([rot.set(dev[0], 2, dev[1], dev[3])], 6, dev[2], "f32")
            rot.backward_device([rot.grad(dev[0], 2, dev[4], dev[5], dev[3], dev[6])], 6, dev[2], "f32")
            y, dx, dw = dev[1].download(), dev[5].download(), dev[6].download()
            for d in dev:
                d.free()
        np.testing.assert_array_equal(y[~live], 7)
        np.testing.assert_array_equal(dx[~live], 0)
        args = dict(norm=64, weight=w, first=48, dims=16)
        want = oracle.heads(x[live], table, positions[live], **args)
        np.testing.assert_allclose(y[live], want, atol=1e-5)
        dx_want, dw_want = oracle.heads_backward(dy[live], x[live], table, positions[live], **args)
        np.testing.assert_allclose(dx[live], dx_want, atol=1e-5)
        np.testing.assert_allclose(dw, dw_want if live.any() else 0, atol=1e-5)


def test_no_tokens(gpu_ctx):
    with HeadRotation(gpu_ctx, 64, 64, 16, table=rotation_table(8, 16)) as rot:
        out = rot.backward(np.zeros((0, 2, 64), np.float32), np.zeros((0, 2, 64), np.float32), np.zeros(0, np.int32))
        np.testing.assert_array_equal(out["dweight"], 0)
        assert rot.apply(np.zeros((0, 2, 64), np.uint16), np.zeros(0, np.int32)).shape == (0, 2, 64)


def test_in_place_and_apart_give_the_same_and_mixed_types_round_once(gpu_ctx):
    rng, table = np.random.default_rng(7), rotation_table(30, 64)
    x, positions = bf16_bits(rng.standard_normal((50, 4, 576)).astype(np.float32)), rng.integers(0, 30, 50).astype(np.int32)
    for norm in (0, 512):
        with HeadRotation(gpu_ctx, 576, norm, 64, 512, "halves", table=table) as rot:
            dev = [gpu_ctx.upload(a) for a in (x, x, positions, np.zeros(x.shape, np.float32), np.zeros(x.shape, np.uint16))]
            rot.apply_device([rot.set(dev[0], 4, dev[0])], 50, dev[2])
            rot.apply_device([rot.set(dev[1], 4, dev[3])], 50, dev[2], "bf16", "f32")
            rot.apply_device([rot.set(dev[1], 4, dev[4])], 50, dev[2])
            in_place, wide, apart = dev[0].download(), dev[3].download(), dev[4].download()
            for d in dev:
                d.free()
        np.testing.assert_array_equal(in_place, apart)
        np.testing.assert_array_equal(apart, bf16_bits(wide))


def test_gradients_are_the_same_on_every_run(gpu_ctx):
    rng, _, table, positions, weight = case_of(700, 9, 128, 128, 0, 128, "halves", "bf16")
    x, dy = (bf16_bits(rng.standard_normal((700, 9, 128)).astype(np.float32)) for _ in range(2))
    with HeadRotation(gpu_ctx, 128, 128, 128, 0, "halves", table=table) as rot:
        a, b = (rot.backward(dy, x, positions, weight) for _ in range(2))
        np.testing.assert_array_equal(a["dx"], b["dx"])
        np.testing.assert_array_equal(a["dweight"], b["dweight"])


def test_host_calls_refuse(gpu_ctx):
    rot = HeadRotation(gpu_ctx, 64, 64, 16, table=rotation_table(8, 16))
    x, pos = np.zeros((3, 2, 64), np.float32), np.zeros(3, np.int32)
    for args in ((x[..., :32], pos), (x[0], pos), (x.astype(np.float64), pos), (x, None), (x, pos[:2]), (x, pos.astype(np.float32)),
                 (x, pos + 8), (x, pos - 2), (x, pos, np.ones(32)), (x, pos, np.ones((64, 1)))):
        with pytest.raises(ValueError):
            rot.apply(*args)
    for dy, other in ((x, x.astype(np.float64)), (x, x[:2]), (bf16_bits(x), x)):
        with pytest.raises(ValueError):
            rot.backward(dy, other, pos)
    rot.close()
    with pytest.raises(RuntimeError):
        rot.apply_device([], 1)
    with pytest.raises(RuntimeError):
        rot.open_gradients()
