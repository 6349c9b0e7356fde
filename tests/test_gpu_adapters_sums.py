"""Adapters whose h = scale (down x) fills all 24 bits of FP32 and whose base cancels it: what is left shows every bit
that a kernel drops between the two products.

All values are chosen so that each product and each partial sum, in any order, is a whole multiple of |scale| below 2^24
of them: three columns of x hold a whole number's bytes, down's factors 2^16, 2^8 and 1 put it together, up picks one rank
per output, and base is minus that plus a small number. So the result, a small number, is exact.
"""

import numpy as np
import pytest

from oracle import adapters as oracle
from oracle.formats import bf16_bits, bf16_values
from vesper_amd.adapters import AdapterBank

pytestmark = pytest.mark.gpu


def digits(rng, width, rank, factor):
    """(columns [rank, 3], down [rank, width]): rank r is factor times the number in its three columns."""
    columns = rng.permutation(width)[:3 * rank].reshape(rank, 3)
    down = np.zeros((rank, width), np.float32)
    down[np.arange(rank)[:, None], columns] = np.float32(factor) * np.array([65536, 256, 1], np.float32)
    return columns, down


def pick(rng, rows, rank, value):
    """up [rows, rank]: +-value at one rank of each output."""
    up = np.zeros((rows, rank), np.float32)
    up[np.arange(rows), rng.integers(0, rank, rows)] = value * rng.choice([-1, 1], rows)
    return up


def run(gpu_ctx, tokens, rows, width, rank, adapters, step, seed):
    """Bytes for x; base = -(the adapter) + small multiples of `step`, the results."""
    rng = np.random.default_rng(seed)
    x = rng.integers(0, 256, (tokens, width)).astype(np.float32)
    ids = rng.integers(-1, 3, tokens).astype(np.int32)   # the last slot is empty
    ids[0] = 0
    sums, _ = oracle.apply(x, ids, np.zeros((tokens, rows)), adapters)
    small = rng.integers(-99, 100, (tokens, rows)) * step
    base = (small - sums).astype(np.float32)
    want = base.astype(np.float64) + sums   # base's own rounding, half of 2 steps at most, is part of the result
    assert np.abs(want).max() <= 101 * step
    with AdapterBank(gpu_ctx, rows, width, 3, rank, tokens) as bank:
        for slot, (down, up, scale) in adapters.items():
            bank.load(slot, bf16_bits(down), bf16_bits(up), scale)
        got = bank.apply(bf16_bits(x), ids, base)
    with_one = ids >= 0
    with_one &= ids < 2
    np.testing.assert_array_equal(bf16_values(got[with_one]), want[with_one])
    np.testing.assert_array_equal(got[~with_one], bf16_bits(base[~with_one]))


# one launch (one and two rank tiles, the second with more of K than its ring holds), two launches (four rank tiles, and
# more in turns; one and two rank tiles of a wide K), the grouped form with one part of K and with several, for every
# count of rank tiles that has a kernel of its own
SHAPES = [(1, 72, 104, 16), (20, 72, 200, 32), (3, 72, 2120, 16), (5, 136, 520, 64), (40, 72, 1544, 256),
          (24, 72, 16384, 16), (17, 72, 7176, 32),
          (150, 72, 104, 16), (150, 72, 264, 32), (150, 200, 264, 64), (150, 72, 520, 128), (150, 328, 776, 256),
          (150, 72, 1544, 16), (170, 72, 1544, 32), (200, 72, 1544, 64), (300, 72, 7176, 64), (300, 72, 7176, 128),
          (150, 72, 1544, 256)]


@pytest.mark.parametrize("tokens,rows,width,rank", SHAPES)
def test_every_bit_of_h_counts(gpu_ctx, tokens, rows, width, rank):
    rng = np.random.default_rng(tokens + rank)
    adapters = {slot: (digits(rng, width, rank, 1)[1], pick(rng, rows, rank, 1), scale)
                for slot, scale in enumerate((1.0, -1.0))}
    run(gpu_ctx, tokens, rows, width, rank, adapters, 1, tokens)


@pytest.mark.parametrize("tokens", [2, 30, 150])
@pytest.mark.parametrize("rank", [16, 64])
def test_the_scale_is_part_of_h(gpu_ctx, tokens, rank):
    """A scale that is no power of two: h is the product rounded once to FP32."""
    rng = np.random.default_rng(rank)
    rows, width, scale = 72, 264, np.float32(1.1)
    columns, down = digits(rng, width, rank, 1)
    up = pick(rng, rows, rank, 1)
    x = rng.integers(0, 256, (tokens, width)).astype(np.float32)
    h = np.float32(scale) * (x @ down.T)   # x @ down.T is whole and exact
    sums = h.astype(np.float64) @ up.T.astype(np.float64)
    base = (rng.integers(-64, 65, (tokens, rows)) * 2.0 - sums).astype(np.float32)
    want = base.astype(np.float64) + sums   # both are multiples of an FP32 step of h: at most 2^25 / 2^24 = 2
    with AdapterBank(gpu_ctx, rows, width, 1, rank, tokens) as bank:
        bank.load(0, bf16_bits(down), bf16_bits(up), float(scale))
        got = bank.apply(bf16_bits(x), np.zeros(tokens, np.int32), base)
    np.testing.assert_array_equal(got, bf16_bits(want.astype(np.float32)))


@pytest.mark.parametrize("tokens,rank", [(2, 16), (30, 64), (150, 16), (150, 64)])
def test_h_up_to_the_largest_float(gpu_ctx, tokens, rank):
    """The largest FP32 value is larger than the largest BF16 value, and a small up brings it back."""
    rng = np.random.default_rng(rank + 1)
    rows, width = 72, 264
    columns, down = digits(rng, width, rank, 2.0 ** 104)
    up = pick(rng, rows, rank, 2.0 ** -100)
    x = np.full((tokens, width), 255, np.float32)
    sums = np.float64(np.finfo(np.float32).max) * up.sum(1)[None].astype(np.float64)   # +-(2^24 - 1) 16
    base = (rng.integers(-99, 100, (tokens, rows)) * 16 - sums).astype(np.float32)
    want = base.astype(np.float64) + sums
    with AdapterBank(gpu_ctx, rows, width, 1, rank, tokens) as bank:
        bank.load(0, bf16_bits(down), bf16_bits(up), 1.0)
        got = bank.apply(bf16_bits(x), np.zeros(tokens, np.int32), base)
    np.testing.assert_array_equal(bf16_values(got), want)
