"""A captured step goes on after larger calls on its context have grown the scratch that it uses, and can be the first step of
its layer: opening a cache reserves what its steps need."""

import ctypes as C

import numpy as np
import pytest

from oracle.formats import bf16_bits
from oracle.projections import fp8_weights
from tests.test_gpu_cached_attention import PAGE, TABLE, options, projections  # noqa: F401 (a fixture)
from tests.test_gpu_row_gemv import projections as single
from tests.test_gpu_scratch import Graph
from vesper_amd import _lib
from vesper_amd.attention import rotation_table
from vesper_amd.projections import NativeProjections

pytestmark = pytest.mark.gpu


def test_a_captured_projection_after_larger_ones(gpu_ctx):
    rng, rows, width, tokens, many = np.random.default_rng(1), 512, 8192, 20, 3000
    w, sw = fp8_weights(rng, rows, width, 32)
    bits = bf16_bits(rng.standard_normal((many, width)).astype(np.float32))
    with single(w, sw, 32) as proj, _lib.Context(0) as ctx:
        x, y = ctx.upload(bits), ctx.empty((many, rows), np.uint16)
        stream = ctx.stream()

        def call(on, n):
            ctx.lib.fp8_projection(ctx._h(), C.c_void_p(proj.tiled["p"]), rows, width, 32, _lib.vp(x), n, _lib.vp(y), None, None,
                                   None, on)
        graph = Graph(ctx, stream, lambda: call(C.c_void_p(stream), tokens))
        graph.launch()
        want = y.download()[:tokens]
        for _ in range(3):
            call(None, many)      # 24 MB of codes: the scratch of the graph would not hold them
            ctx.sync()
            junk = ctx.upload(np.full(1 << 22, 0xFF, np.uint8))
            y.upload(np.zeros((many, rows), np.uint16))
            ctx.sync()
            graph.launch()
            np.testing.assert_array_equal(y.download()[:tokens], want)
            junk.free()
        graph.close()
        call(None, tokens)
        np.testing.assert_array_equal(y.download()[:tokens], want)
        ctx.destroy_stream(stream)


def test_a_first_step_is_captured_and_replayed_between_prompts(projections):  # noqa: F811
    """Decoding captured before anything ran on the context, then a prompt of 1100 tokens through a second layer between any
    two replays: as eager steps of a runtime of its own."""
    rng, table, many = np.random.default_rng(2), rotation_table(1200, 64), 1100
    opened = options(rng, max_tokens=4)
    pages = np.arange(3, dtype=np.int32)[:, None]
    with NativeProjections(projections.arrays) as proj, \
            projections.open_cache(3, PAGE, TABLE, **opened) as eager, \
            proj.open_cache(3, PAGE, TABLE, **opened) as layer:
        ctx = proj.ctx
        x = np.zeros((3, 5120), np.uint16)
        dev = [ctx.upload(a) for a in (x, np.zeros(3, np.int32), np.zeros(3, np.int64), pages, np.zeros(3, np.int32), x)]
        ptr = [d.ptr for d in dev]
        stream = ctx.stream()
        graph = Graph(ctx, stream, lambda: layer.step_device(ptr[0], 3, ptr[1], ptr[2], ptr[3], 1, ptr[4], 3, ptr[5], stream=stream))
        prompt = proj.open_cache(-(-many // 64), 64, table, max_tokens=many, max_batch=1)
        long_x = bf16_bits(rng.standard_normal((many, 5120)).astype(np.float32))
        prompts = []
        for at in range(3):
            x = bf16_bits(rng.standard_normal((3, 5120)).astype(np.float32))
            place = np.full(3, at)
            slots = pages[:, 0].astype(np.int64) * PAGE + at
            for d, a in zip(dev, (x, place.astype(np.int32), slots, pages, (place + 1).astype(np.int32))):
                d.upload(a)
            ctx.sync()
            graph.launch()
            np.testing.assert_array_equal(dev[5].download(), eager.step(x, place, slots, pages, place + 1))
            prompts.append(prompt.step(long_x, np.arange(many), np.arange(many), np.arange(-(-many // 64))[None], np.array([many])))
            np.testing.assert_array_equal(prompts[0], prompts[-1])
        graph.close()
        ctx.destroy_stream(stream)
        for d in dev:
            d.free()


def test_reserved_calls_fit(gpu_ctx):
    """After a reserve, calls of any number of tokens up to its own can be captured on a fresh context, where they could not
    allocate: decode shapes whose sums are split, GEMMs of few and of many tokens."""
    rng = np.random.default_rng(3)
    for rows, width, most, counts in ((64, 65536, 40, (1, 5, 16, 32, 33, 40)), (512, 8192, 700, (32, 128, 129, 700))):
        w, sw = fp8_weights(rng, rows, width, 32)
        with single(w, sw, 32) as proj, _lib.Context(0) as ctx:
            x, y = ctx.upload(bf16_bits(rng.standard_normal((most, width)).astype(np.float32))), ctx.empty((most, rows), np.uint16)
            ctx.lib.fp8_reserve(ctx._h(), rows, width, most)
            stream = ctx.stream()
            for n in counts:
                def call(on, at):
                    at.lib.fp8_projection(at._h(), C.c_void_p(proj.tiled["p"]), rows, width, 32, _lib.vp(x), n, _lib.vp(y), None, None,
                                          None, on)
                graph = Graph(ctx, stream, lambda: call(C.c_void_p(stream), ctx))
                graph.launch()
                got = y.download()[:n]
                graph.close()
                call(None, gpu_ctx)
                gpu_ctx.sync()
                np.testing.assert_array_equal(y.download()[:n], got)
            for bad in ((rows + 32, width, 1), (rows, width + 64, 1), (rows, width, -1), (rows, width, 2 ** 20 + 1)):
                with pytest.raises(ValueError):
                    ctx.lib.fp8_reserve(ctx._h(), *bad)
            ctx.destroy_stream(stream)
