"""Large calls take several heads of a token at once; a row's values do not depend on what is beside it, so they are the small
calls' bit for bit."""

import numpy as np
import pytest

from oracle.formats import bf16_bits
from vesper_amd.attention import HeadRotation, rotation_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,norm,dims,style,tokens", [(64, 64, 32, "halves", 19000), (128, 128, 128, "halves", 9500), (192, 0, 64, "pairs", 4800),
                                                          (512, 512, 64, "pairs", 2400), (128, 64, 64, "pairs", 9500)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_calls_are_the_small_ones(gpu_ctx, width, norm, dims, style, tokens, dtype):
    rng = np.random.default_rng(width + norm)
    heads, small = (5, 2), 100   # neither a multiple of four
    positions = rng.integers(-1, 50, tokens).astype(np.int32)
    with HeadRotation(gpu_ctx, width, norm=norm, dims=dims, style=style, table=rotation_table(50, dims)) as rot:
        def rows(h):
            x = rng.standard_normal((tokens, h, width)).astype(np.float32)
            return bf16_bits(x) if dtype == "bf16" else x
        x = [rows(h) for h in heads]
        weights = [(rng.random(norm) + 0.5).astype(np.float32) if norm else None for _ in heads]
        dev = [gpu_ctx.upload(a) for a in x]
        dev_w = [None if w is None else gpu_ctx.upload(w) for w in weights]
        at = gpu_ctx.upload(positions)
        rot.apply_device([rot.set(d, h, d, w) for d, h, w in zip(dev, heads, dev_w)], tokens, at, dtype)   # in place
        got = [d.download() for d in dev]
        for i in range(2):
            for first in rng.integers(0, tokens - small, 5):
                part = slice(first, first + small)
                want = rot.apply(x[i][part], positions[part] if dims else None, weights[i])
                np.testing.assert_array_equal(got[i][part], want)
        for d in dev + dev_w + [at]:
            if d is not None:
                d.free()


@pytest.mark.parametrize("width,dtype,tokens", [(64, "f32", 30000), (128, "bf16", 20000), (512, "f32", 3000)])
def test_many_turns_of_the_gradients(gpu_ctx, width, dtype, tokens):
    """Workgroups go over several rows: dx is the small calls', and dweight their sum. A column's sum is a chain of a lane's
    rows, at most 32 lanes, ten parts and two trees of at most 16; in a small call as many but for one row a lane. So both are
    within 2^-24 (rows a lane + 2 * 80) of the terms' magnitudes |g u| <= (g^2 + u^2) / 2, which are 1 on average here (at
    most 1.1 over 9,000 rows and more)."""
    rng = np.random.default_rng(width)
    heads, small = 3, 250
    x = rng.standard_normal((tokens, heads, width)).astype(np.float32)
    dy = rng.standard_normal((tokens, heads, width)).astype(np.float32)
    if dtype == "bf16":
        x, dy = bf16_bits(x), bf16_bits(dy)
    positions = rng.integers(-1, 40, tokens)
    weight = (rng.random(width) + 0.5).astype(np.float32)
    with HeadRotation(gpu_ctx, width, norm=width, dims=32, table=rotation_table(40, 32)) as rot:
        got = rot.backward(dy, x, positions, weight)
        total = np.zeros(width)
        for first in range(0, tokens, small):
            part = slice(first, first + small)
            one = rot.backward(dy[part], x[part], positions[part], weight)
            np.testing.assert_array_equal(got["dx"][part], one["dx"])
            total += one["dweight"]
        turns = -(-tokens * heads // (1280 * 256 // (width // 8)))
        assert np.all(np.abs(got["dweight"] - total) <= 2.0 ** -24 * (turns + 160) * 1.1 * tokens * heads)
