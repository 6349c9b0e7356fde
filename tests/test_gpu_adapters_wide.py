"""Adapters at the widths of the framework's projections: the kernels, parts of K and rounds that only a long row reaches.

Small integers, at most 1600 columns of x not zero: every partial sum is a multiple of 1/2 below 2^23, so every result is
the oracle's, rounded once. The workspace starts as NaN, so a part that no one wrote shows."""

import numpy as np
import pytest

from oracle import adapters as oracle
from oracle.formats import bf16_bits, bf16_values
from vesper_amd.adapters import AdapterBank
from vesper_amd.dispatch import ExpertDispatch

pytestmark = pytest.mark.gpu


def integers(rng, lo, hi, shape):
    return rng.integers(lo, hi + 1, shape, np.int8).astype(np.float32)


def make(rng, rows, width, rank):
    return integers(rng, -2, 2, (rank, width)), integers(rng, -2, 2, (rows, rank))


def fill(ctx, bank, pairs, scales, slots):
    """Slot s <- pair s % len(pairs) with scale scales[s % len(scales)]; {slot: adapter} for the oracle."""
    dev = [[ctx.upload(bf16_bits(a)) for a in pair] for pair in pairs]
    adapters = {}
    for s in range(slots):
        down, up = pairs[s % len(pairs)]
        adapters[s] = (down, up, scales[s % len(scales)])
        bank.load_device(s, *dev[s % len(pairs)], len(down), adapters[s][2])
    ctx.sync()
    for pair in dev:
        for a in pair:
            a.free()
    return adapters


def run(ctx, bank, ids, adapters, seed, dtype="bf16", plans=(False,)):
    rng = np.random.default_rng(seed)
    tokens, rows, width = len(ids), bank.rows, bank.width
    x = np.zeros((tokens, width), np.float32)
    columns = rng.permutation(width)[:1600]
    x[:, columns] = integers(rng, -2, 2, (tokens, len(columns)))
    base = integers(rng, -99, 99, (tokens, rows))
    narrow = {s: (down[:, columns], up, scale) for s, (down, up, scale) in adapters.items() if s in ids}
    want = bf16_bits(oracle.apply(x[:, columns], ids, base, narrow)[0].astype(np.float32))
    dev = [ctx.upload(a) for a in (bf16_bits(x), ids.astype(np.int32), base if dtype == "f32" else bf16_bits(base))]
    with ExpertDispatch(ctx, bank.slots, 1, tokens) as d:
        d.plan_device(dev[1], tokens)
        for planned in plans:
            y = ctx.upload(np.zeros((tokens, rows), np.uint16))
            ctx.copy_h2d(bank.workspace, np.full(bank.workspace_bytes // 4, 0x7FC07FC0, np.uint32))
            bank.apply_device(dev[0], dev[1], tokens, dev[2], y, dtype, plan=d.plan if planned else None)
            np.testing.assert_array_equal(y.download(), want, err_msg=f"plan {planned}")
            y.free()
    for a in dev:
        a.free()


# few tokens: one launch whose ring goes round, two launches of one, two and more rank tiles, up to 32 parts of K;
# the grouped form with up to 32 parts
@pytest.mark.parametrize("tokens,width,rank", [
    (1, 7176, 16), (1, 5120, 12), (16, 7176, 16), (40, 3080, 16), (20, 2056, 32),
    (1, 16384, 16), (24, 16384, 16), (128, 16384, 16), (1, 7176, 32), (24, 7176, 32), (128, 16384, 32),
    (1, 16384, 64), (24, 16384, 64), (128, 16376, 64), (33, 16384, 128), (64, 7176, 256),
    (150, 16384, 16), (600, 16384, 16), (150, 16384, 32), (1000, 16384, 32), (200, 16384, 64), (1000, 16376, 64),
    (150, 16384, 128), (600, 7176, 128), (70, 16384, 256), (1000, 16384, 256), (3700, 7176, 40)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_wide_rows(gpu_ctx, tokens, width, rank, dtype):
    rng = np.random.default_rng(tokens + rank)
    with AdapterBank(gpu_ctx, 328, width, 4, rank, tokens) as bank:
        adapters = fill(gpu_ctx, bank, [make(rng, 328, width, r) for r in (rank, max(1, rank - 7), rank)], (1.0, -2.0, 0.5), 3)
        ids = rng.integers(-1, 4, tokens)
        ids[0] = 0
        run(gpu_ctx, bank, ids, adapters, rank, dtype, (False, True))


@pytest.mark.parametrize("tokens,width,rank,slots", [(1000, 7176, 16, 200), (1000, 7176, 64, 200), (600, 7176, 24, 90),
                                                     (1000, 2056, 16, 600), (1000, 2056, 64, 600), (1000, 2056, 256, 200),
                                                     (300, 7176, 100, 150)])
def test_more_tiles_than_the_split_of_k_leaves_room_for(gpu_ctx, tokens, width, rank, slots):
    """The tiles that the tokens make reduce the parts of K on the device, down to one, which stays a sum all the same."""
    rng = np.random.default_rng(slots + rank)
    with AdapterBank(gpu_ctx, 72, width, slots, rank, tokens) as bank:
        adapters = fill(gpu_ctx, bank, [make(rng, 72, width, r) for r in (rank, max(1, rank // 2), rank)], (1.0, -2.0, 0.5, -1.0),
                        slots)
        run(gpu_ctx, bank, rng.permutation(np.arange(tokens) % slots), adapters, rank, "f32", (False, True))


@pytest.mark.parametrize("tokens", [4095, 4096, 4097])
@pytest.mark.parametrize("rank", [16, 64])
def test_around_the_most_tokens_that_down_counts_itself(gpu_ctx, tokens, rank):
    rng = np.random.default_rng(tokens)
    with AdapterBank(gpu_ctx, 72, 1544, 5, rank, tokens) as bank:
        adapters = fill(gpu_ctx, bank, [make(rng, 72, 1544, rank - s) for s in range(3)], (1.0, -2.0, 0.5), 4)
        run(gpu_ctx, bank, rng.integers(-1, 5, tokens), adapters, rank, plans=(False, True))


@pytest.mark.parametrize("tokens,rows,width,rank", [(2400, 1032, 16384, 64), (2400, 1032, 16384, 32), (4200, 3592, 7176, 64)])
def test_calls_larger_than_the_caches(gpu_ctx, tokens, rows, width, rank):
    """x, base and y of more than 80 MiB: x is read past the caches."""
    rng = np.random.default_rng(rows)
    with AdapterBank(gpu_ctx, rows, width, 3, rank, tokens) as bank:
        adapters = fill(gpu_ctx, bank, [make(rng, rows, width, rank - 9 * s) for s in range(3)], (1.0, -2.0, 0.5), 3)
        run(gpu_ctx, bank, rng.integers(-1, 3, tokens), adapters, rank, plans=(False, True))


@pytest.mark.parametrize("tokens", [1, 24, 200])
def test_random_values_of_a_wide_projection(gpu_ctx, tokens):
    """Unit-variance x, weights as a fine-tune has them. An FP32 chain of n additions is within n 2^-24 of the terms'
    magnitudes: at most width / 32 + rank / 8 matrix steps and 50 additions, counted twice for what a matrix step rounds
    inside; a BF16 result is within 2^-8 of its value."""
    rng = np.random.default_rng(tokens)
    rows, width, rank = 264, 16384, 64
    down = bf16_values(bf16_bits(rng.standard_normal((rank, width)).astype(np.float32)))
    up = bf16_values(bf16_bits((rng.standard_normal((rows, rank)) / np.sqrt(width * rank)).astype(np.float32)))
    x = bf16_bits(rng.standard_normal((tokens, width)).astype(np.float32))
    base = rng.standard_normal((tokens, rows)).astype(np.float32)
    with AdapterBank(gpu_ctx, rows, width, 1, rank, tokens) as bank:
        bank.load(0, bf16_bits(down), bf16_bits(up), 0.75)
        got = bf16_values(bank.apply(x, np.zeros(tokens, np.int32), base)).astype(np.float64)
    want, size = oracle.apply(bf16_values(x), np.zeros(tokens, int), base, {0: (down, up, 0.75)})
    steps = width / 32 + rank / 8 + 50
    limit = np.abs(want) * 2.0 ** -8 + (1 + 2.0 ** -8) * size * 2 * steps * 2.0 ** -24
    assert np.all(np.abs(got - want) <= limit)
