"""The 4-bit paged cache and its attention on the device against the 64-bit oracle.

Codes and scales are the definition's, whatever the size of a call: compared bit for bit on keys that are stored as they
are. Attention: a probability is rounded to BF16 (2^-8 of it), the result once more (2^-8 of it); a logit is a chain of at
most 48 matrix steps and 8 roundings of terms whose magnitudes are bounded by the oracle's, and an error d of a logit changes
its probability and the sum by d of them each."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_round, bf16_values
from tests.test_gpu_scratch import Graph
from vesper_amd import _lib
from vesper_amd.attention import HeadRotation, KVCache4, rotation_table

pytestmark = pytest.mark.gpu
KINDS = {"64": (64, None), "128": (128, None), "256": (256, None), "512": (512, 512), "576": (576, 512)}


def open_cache(ctx, kind, pages, page, heads, query_heads, max_tokens=4096, max_batch=256):
    width, value_width = KINDS[kind]
    return KVCache4(ctx, pages, page, heads, width, value_width, query_heads=query_heads, max_tokens=max_tokens, max_batch=max_batch)


def stored(cache, which="k"):
    """(codes 0-15 [pages * page, heads, width], scales) of the whole cache, by slot."""
    raw = cache.read(range(cache.pages))
    width = cache.width if which == "k" else cache.value_width
    flat = lambda a: a.transpose(0, 2, 1, 3).reshape(cache.pages * cache.page, cache.heads, -1)  # noqa: E731
    return oracle.unpack(flat(raw[which + "_codes"])), flat(raw[which + "_scales"])[..., :width // 32]


# -- append ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,page,heads", [(1, 16, 1), (37, 16, 3), (200, 64, 2), (5, 1024, 8)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_as_they_are(gpu_ctx, kind, tokens, page, heads, dtype):
    rng = np.random.default_rng(tokens + heads)
    pages = -(-tokens // page) + 2
    with open_cache(gpu_ctx, kind, pages, page, heads, heads) as cache:
        def rows(width):
            x = (rng.standard_normal((tokens, heads, width)) * np.exp2(rng.integers(-25, 60, (tokens, heads, 1)))).astype(np.float32)
            x[0, 0, :32] = np.resize(np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 6, -0.25, -0.0]), 32)
            x[-1, -1, 32:64] = 0
            return bf16_bits(x) if dtype == "bf16" else x
        k, v = rows(cache.width), rows(cache.value_width) if cache.apart else None
        slots = rng.permutation(pages * page)[:tokens]
        slots[tokens // 2] = slots[tokens // 2] if tokens < 3 else -1
        got = cache.append(k, slots, v)
        for name, x in (("k", k), ("v", v)):
            if x is None:
                continue
            codes, scales = oracle.encode(bf16_values(x) if dtype == "bf16" else bf16_round(x))
            live = slots >= 0
            have = stored(cache, name)
            np.testing.assert_array_equal(have[0][slots[live]], codes[live])
            np.testing.assert_array_equal(have[1][slots[live]], scales[live])
            np.testing.assert_array_equal(bf16_values(got[name])[live], oracle.decode(codes, scales)[live])
            np.testing.assert_array_equal(got[name][~live], 0)


def test_append_of_what_is_not_finite(gpu_ctx):
    x = np.ones((3, 1, 512), np.float32)
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 500] = np.inf, np.nan, 3.39e38
    with open_cache(gpu_ctx, "512", 1, 16, 1, 1) as cache:
        got = bf16_values(cache.append(x, np.arange(3))["k"])
        codes, scales = oracle.encode(bf16_round(x))
        np.testing.assert_array_equal(stored(cache)[1][:3], scales)
        np.testing.assert_array_equal(stored(cache)[0][:3], codes)
        np.testing.assert_array_equal(got, oracle.decode(codes, scales))


@pytest.mark.parametrize("kind,heads,norm,dims,style", [("512", 1, 512, 64, "pairs"), ("576", 1, 512, 64, "pairs"), ("128", 8, 128, 128, "halves"),
                                                        ("64", 2, 0, 64, "halves"), ("256", 3, 256, 0, "pairs")])
@pytest.mark.parametrize("lead", [0, 1])
def test_append_is_heads_then_append(gpu_ctx, kind, heads, norm, dims, style, lead):
    """Normalized and rotated on the way: the codes of HeadRotation's BF16 result, bit for bit, of strided rows too."""
    rng, tokens, page = np.random.default_rng(heads + norm + lead), 70, 16
    width = KINDS[kind][0]
    table, positions = rotation_table(99, dims) if dims else None, rng.integers(0, 99, tokens).astype(np.int32)
    weight = rng.uniform(.5, 1.5, norm).astype(np.float32) if norm else None
    with open_cache(gpu_ctx, kind, 9, page, heads, heads) as cache, \
            HeadRotation(gpu_ctx, width, norm, dims, style=style, table=table) as rot:
        stride = heads * width + (8 if not lead else 3)
        raw = bf16_bits(rng.standard_normal((tokens, stride)).astype(np.float32))
        x = raw[:, lead:lead + heads * width].reshape(tokens, heads, width)
        v = bf16_bits(rng.standard_normal((tokens, heads, width)).astype(np.float32)) if cache.apart else None
        slots = rng.permutation(9 * page)[:tokens].astype(np.int64)
        slots[3], slots[9], positions[20] = -5, 9 * page, 99 if dims else 0
        live = np.ones(tokens, bool)
        live[[3, 9]] = False
        live[20] = not dims
        turned = rot.apply(np.ascontiguousarray(x[live]), positions[live] if dims else None, weight)
        dev = [None if a is None else gpu_ctx.upload(a) for a in (raw, v, slots, positions, weight, np.full(x.shape, 7, np.uint16))]
        cache.append_device(dev[0].ptr + 2 * lead, dev[2], tokens, dev[1], rot, dev[3], dev[4], k_stride=stride, k_rounded_ptr=dev[5])
        rounded = dev[5].download()
        for d in dev:
            if d is not None:
                d.free()
        codes, scales = oracle.encode(bf16_values(turned))
        have = stored(cache)
        np.testing.assert_array_equal(have[0][slots[live]], codes)
        np.testing.assert_array_equal(have[1][slots[live]], scales)
        np.testing.assert_array_equal(bf16_values(rounded[live]), oracle.decode(codes, scales))
        np.testing.assert_array_equal(rounded[~live], 7)


# -- attend ------------------------------------------------------------------------------------------------

def fill(cache, rng, table, lengths, nan_tokens=()):
    """Random codes and scales in every sequence's tokens; (keys, values) [B][length][heads][...] float64. nan_tokens
    (b, token): NaN in a block of the values, or of a latent's last."""
    tokens = int(lengths.sum())
    slots = np.concatenate([table[b][np.arange(n) // cache.page].astype(np.int64) * cache.page + np.arange(n) % cache.page
                            for b, n in enumerate(lengths)] or [np.zeros(0, np.int64)])

    def rows(width):
        x = rng.standard_normal((tokens, cache.heads, width)) * np.exp2(rng.integers(-2, 2, (tokens, cache.heads, width // 32))).repeat(32, -1)
        return bf16_round(x.astype(np.float32))
    k, v = rows(cache.width), rows(cache.value_width) if cache.apart else None
    first = np.concatenate([[0], np.cumsum(lengths)])
    for b, at in nan_tokens:
        (v if cache.apart else k)[first[b] + at, :, 40] = np.nan
    for at in range(0, tokens, 1 << 16):
        part = slice(at, at + (1 << 16))
        cache.append(k[part], slots[part], None if v is None else v[part])
    kd = oracle.decode(*oracle.encode(k))
    vd = kd[..., :cache.value_width] if v is None else oracle.decode(*oracle.encode(v))
    return [kd[first[b]:first[b + 1]] for b in range(len(lengths))], [vd[first[b]:first[b + 1]] for b in range(len(lengths))]


def pages_for(rng, lengths, page, spare=2, columns=None):
    held = -(-lengths // page)
    order = rng.permutation(int(held.sum()) + spare).astype(np.int32)
    table = np.full((len(lengths), columns or max(int(held.max(initial=0)), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order)


def check(got, q, keys, lengths, scale, want, lse, size):
    """Within the header's bounds; exactly zero and -infinity where a row sees nothing."""
    group = q.shape[1] // (keys[0].shape[1] if keys else 1)
    largest = max((np.abs(k).max(initial=0.0, axis=(0, 1)) for k in keys), key=lambda a: a.sum(), default=np.zeros(1))
    s = np.abs(q).astype(np.float64) @ np.maximum.reduce([np.abs(k).max(initial=0.0, axis=(0, 1)) for k in keys] or [largest]) * scale
    d = (56 * 2.0 ** -24 * s + 2.0 ** -22)[..., None]     # of a logit, and of the power of two
    limit = 2.0 ** -8 * (1 + 2.0 ** -8) * size + 2 * d * size + 2.0 ** -8 * np.abs(want) + 1e-30
    out = bf16_values(got["out"]).astype(np.float64)
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(out), nan)
    worst = np.max(np.where(nan, -1, np.abs(out - want) - limit), initial=-1)
    assert worst <= 0, f"{worst:.3e} past the limit"
    empty = np.isneginf(lse)
    np.testing.assert_array_equal(np.isneginf(got["lse"]), empty)
    np.testing.assert_array_equal(np.isnan(got["lse"]), np.isnan(lse))
    np.testing.assert_array_equal(out[empty], 0)
    rest = ~empty & ~np.isnan(lse)
    assert np.all(np.abs(got["lse"][rest] - lse[rest]) <= d[rest, 0] + 2.0 ** -22 * (1 + np.abs(lse[rest])) + 64 * 2.0 ** -24)


# (kind, query heads, key heads, lengths, counts (None: one each), page, window, sinks)
ATTENDS = [
    ("512", 64, 1, [1], None, 64, 0, False), ("512", 64, 1, [300], None, 64, 0, True), ("512", 64, 1, [33, 0, 1, 64, 129], None, 16, 0, True),
    ("576", 128, 1, [77, 200], None, 32, 0, False), ("576", 16, 1, [500, 31, 32], None, 64, 0, False), ("576", 5, 1, [65], None, 64, 0, True),
    ("512", 64, 1, [70, 9], [4, 4], 16, 0, True), ("576", 128, 1, [40], [3], 16, 0, False), ("512", 8, 1, [90, 40], [17, 40], 32, 0, False),
    ("128", 32, 8, [1, 500, 33], None, 16, 0, False), ("128", 8, 8, [257, 64], None, 128, 0, True), ("128", 40, 8, [100], [100], 16, 0, False),
    ("64", 14, 2, [129, 2], None, 16, 0, True), ("64", 14, 2, [150, 60], [150, 7], 64, 0, False), ("64", 71, 1, [200], [2], 16, 0, False),
    ("256", 8, 2, [130, 31], None, 32, 0, False), ("256", 16, 1, [70], [20], 16, 0, True),
    ("512", 64, 1, [300, 20, 129], [5, 20, 1], 128, 16, True), ("128", 32, 8, [400, 128, 127], None, 16, 128, False),
    ("64", 4, 4, [90], [90], 16, 1, False), ("576", 16, 1, [200, 31], [60, 31], 16, 33, False),
    ("128", 16, 4, [3, 0, 2, 5], [4, 2, 2, 1], 16, 0, True),           # more rows than tokens: the first see nothing
    ("64", 8, 1, [10, 300, 20], [0, 3, 1], 16, 0, False), ("512", 16, 1, [50, 8], [0, 8], 16, 0, False),
]


@pytest.mark.parametrize("kind,heads,kv_heads,lengths,counts,page,window,sinks", ATTENDS)
def test_attend(gpu_ctx, kind, heads, kv_heads, lengths, counts, page, window, sinks):
    rng = np.random.default_rng(heads + sum(lengths))
    lengths = np.array(lengths)
    n = np.ones(len(lengths), int) if counts is None else np.array(counts)
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round((rng.standard_normal((int(n.sum()), heads, cache.width)) * 2).astype(np.float32))
        s = (rng.standard_normal(heads) * 2).astype(np.float32) if sinks else None
        scale = cache.width ** -0.5
        want = oracle.attend(q, keys, values, lengths, n, scale, window, s)
        check(cache.attend(bf16_bits(q), table, lengths, scale, counts, window, s), q, keys, lengths, scale, *want)


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("576", 16, 1), ("128", 32, 8), ("64", 4, 4), ("256", 8, 2)])
@pytest.mark.parametrize("length", [1, 31, 1000, 20011])
def test_equal_logits_give_the_mean(gpu_ctx, kind, heads, kv_heads, length):
    """q = 0: every probability is 1, so every sum is exact (multiples of 1/2 below 2^23) and the mean is rounded twice."""
    rng, page = np.random.default_rng(length), 64
    table, pages = pages_for(rng, np.array([length]), page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        grid = np.concatenate([oracle.GRID, -oracle.GRID[1:]])
        draw = lambda w: rng.choice(grid, (length, kv_heads, w)).astype(np.float32)  # noqa: E731
        k, v = draw(cache.width), draw(cache.value_width) if cache.apart else None
        for x in (k, v):
            if x is not None:
                x[..., ::32] = 6            # one scale for every block
        slots = table[0][np.arange(length) // page].astype(np.int64) * page + np.arange(length) % page
        cache.append(k, slots, v)
        got = cache.attend(np.zeros((1, heads, cache.width), np.uint16), table, np.array([length]), 1.0)
        mean = (k[..., :cache.value_width] if v is None else v).sum(0, dtype=np.float64) / length
        want = np.repeat(mean, heads // kv_heads, 0)[None]
        assert np.all(np.abs(bf16_values(got["out"]) - want) <= 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -12))
        np.testing.assert_allclose(got["lse"], np.log(length), rtol=2.0 ** -21, atol=2.0 ** -23)


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("128", 32, 8), ("64", 4, 2)])
def test_many_sequences_of_all_lengths(gpu_ctx, kind, heads, kv_heads):
    """More work than the device has units, so that sequences share and are shared by them."""
    rng, page = np.random.default_rng(3), 16
    lengths = np.array([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129] * 8 + [1500, 900, 0, 3])
    lengths = rng.permutation(lengths)
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round((rng.standard_normal((len(lengths), heads, cache.width)) * 2).astype(np.float32))
        some = heads // kv_heads * np.arange(kv_heads)          # the oracle on one head of each key head
        want = oracle.attend(q[:, some], keys, values, lengths, [1] * len(lengths), 0.1)
        got = cache.attend(bf16_bits(q), table, lengths, 0.1)
        check({k: a[:, some] for k, a in got.items()}, q[:, some], keys, lengths, 0.1, *want)


@pytest.mark.parametrize("kind,heads,kv_heads,count", [("512", 64, 1, 1), ("576", 8, 1, 2), ("128", 32, 8, 1), ("64", 6, 2, 5)])
def test_one_long_sequence_beside_short_ones(gpu_ctx, kind, heads, kv_heads, count):
    rng, page = np.random.default_rng(4), 256
    lengths = np.array([7, 70001, 300])
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round((rng.standard_normal((3 * count, heads, cache.width)) * 4).astype(np.float32))
        some = heads // kv_heads * np.arange(kv_heads)
        scale = cache.width ** -0.5
        want = oracle.attend(q[:, some], keys, values, lengths, [count] * 3, scale)
        got = cache.attend(bf16_bits(q), table, lengths, scale)
        check({k: a[:, some] for k, a in got.items()}, q[:, some], keys, lengths, scale, *want)


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 16, 1), ("576", 64, 1), ("128", 16, 4), ("256", 2, 1)])
def test_nan_reaches_those_who_see_it_and_nobody_else(gpu_ctx, kind, heads, kv_heads):
    """NaN tokens behind a sequence's end, before its window, and behind a row of its own sequence."""
    rng, page = np.random.default_rng(8), 16
    held, lengths = np.array([90, 50, 64]), np.array([70, 50, 64])
    counts, window = np.array([3, 6, 2]), 40
    nan = [(0, 70), (0, 89), (0, 10), (1, 48), (2, 3), (2, 22)]
    table, pages = pages_for(rng, held, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, held, nan)
        q = bf16_round(rng.standard_normal((11, heads, cache.width)).astype(np.float32))
        for w in (window, 0):
            want = oracle.attend(q, [k[:n] for k, n in zip(keys, lengths)], [v[:n] for v, n in zip(values, lengths)], lengths, counts, 0.1, w)
            finite = [np.nan_to_num(k) for k in keys]
            check(cache.attend(bf16_bits(q), table, lengths, 0.1, counts, w), q, finite, lengths, 0.1, *want)
            assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()


def test_queries_that_are_not_finite_stay_with_their_row(gpu_ctx):
    rng = np.random.default_rng(9)
    table, pages = pages_for(rng, np.array([100]), 16)
    with open_cache(gpu_ctx, "512", pages, 16, 1, 8) as cache:
        keys, values = fill(cache, rng, table, np.array([100]))
        q = bf16_round(rng.standard_normal((1, 8, 512)).astype(np.float32))
        want = oracle.attend(q, keys, values, [100], [1], 0.05)
        q[0, 2, 77], q[0, 5, 500] = np.nan, np.inf
        got = cache.attend(bf16_bits(q), table, np.array([100]), 0.05)
        assert np.isnan(bf16_values(got["out"][0, [2, 5]])).all() and np.isnan(got["lse"][0, [2, 5]]).all()
        rest = [0, 1, 3, 4, 6, 7]
        check({k: a[:, rest] for k, a in got.items()}, q[:, rest], keys, [100], 0.05, *(a[:, rest] for a in want))


@pytest.mark.parametrize("q_exp,k_exp", [(-60, 40), (60, -20), (-120, 0), (100, -10), (-30, 90)])
def test_magnitudes_of_all_sizes(gpu_ctx, q_exp, k_exp):
    """Queries and keys far from 1, and blocks of a query far from each other."""
    rng = np.random.default_rng(10)
    table, pages = pages_for(rng, np.array([77]), 16)
    with open_cache(gpu_ctx, "128", pages, 16, 2, 8) as cache:
        k = bf16_round((rng.standard_normal((77, 2, 128)) * 2.0 ** max(k_exp, -12)).astype(np.float32))
        v = bf16_round(rng.standard_normal((77, 2, 128)).astype(np.float32))
        slots = table[0][np.arange(77) // 16].astype(np.int64) * 16 + np.arange(77) % 16
        cache.append(k, slots, v)
        q = rng.standard_normal((1, 8, 128)) * 2.0 ** q_exp
        q[:, :4, 32:64] *= 2.0 ** -9
        q = bf16_round(q.astype(np.float32))
        kd, vd = oracle.decode(*oracle.encode(k)), oracle.decode(*oracle.encode(v))
        scale = float(2.0 ** min(max(-q_exp - max(k_exp, -12) - 3, -100), 100))
        want = oracle.attend(q, [kd], [vd], [77], [1], scale)
        check(cache.attend(bf16_bits(q), table, np.array([77]), scale), q, [kd], [77], scale, *want)


def test_large_logits(gpu_ctx):
    """Logits of some thousands: one token takes all, and the running maximum rises again and again."""
    rng = np.random.default_rng(11)
    table, pages = pages_for(rng, np.array([600]), 16)
    with open_cache(gpu_ctx, "64", pages, 16, 1, 4) as cache:
        keys, values = fill(cache, rng, table, np.array([600]))
        q = bf16_round((rng.standard_normal((1, 4, 64)) * 200).astype(np.float32))
        want = oracle.attend(q, keys, values, [600], [1], 1.0)
        got = cache.attend(bf16_bits(q), table, np.array([600]), 1.0)
        check(got, q, keys, [600], 1.0, *want)


def test_pages_outside_the_cache_and_rows_behind_the_last_sequence(gpu_ctx):
    """Bad page numbers hide their tokens, a length past the table's columns is cut; rows that no sequence has stay."""
    rng, page = np.random.default_rng(12), 16
    lengths = np.array([100, 64])
    table, pages = pages_for(rng, lengths, page, columns=7)
    with open_cache(gpu_ctx, "128", pages, page, 2, 4) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round(rng.standard_normal((6, 4, 128)).astype(np.float32))
        first, bad = np.array([0, 1, 3], np.int32), table.copy()
        bad[0, 2], bad[0, 5], bad[1, 0] = pages, -1, 2 ** 31 - 1
        hidden = [np.isin(np.arange(100) // 16, [2, 5]), np.arange(64) // 16 == 0]
        dev = [gpu_ctx.upload(a) for a in (bf16_bits(q), bad, np.array([100, 64], np.int32), first, np.full((6, 4, 128), 7, np.uint16), np.full((6, 4), 7, np.float32))]
        cache.attend_device(dev[0], 6, dev[1], 7, dev[2], 2, dev[4], 0.1, dev[3], lse_ptr=dev[5])
        got = {"out": dev[4].download(), "lse": dev[5].download()}
        np.testing.assert_array_equal(got["out"][3:], 7)
        np.testing.assert_array_equal(got["lse"][3:], 7)
        want = oracle.attend(q[:3], keys, values, lengths, [1, 2], 0.1, hidden=hidden)
        check({k: a[:3] for k, a in got.items()}, q[:3], keys, lengths, 0.1, *want)
        # one row each of two sequences; the first claims more tokens than its table holds, its row none of which it sees
        dev[2].upload(np.array([7 * 16 + 5, -3], np.int32))
        dev[1].upload(np.where(np.arange(7) < 4, table, -1).astype(np.int32))
        cache.attend_device(dev[0], 2, dev[1], 7, dev[2], 2, dev[4], 0.1, lse_ptr=dev[5])
        got = {"out": dev[4].download()[:2], "lse": dev[5].download()[:2]}
        want = oracle.attend(q[:1], [keys[0][:64]], [values[0][:64]], [64], [1], 0.1)
        check({k: a[:1] for k, a in got.items()}, q[:1], [keys[0][:64]], [64], 0.1, *want)
        np.testing.assert_array_equal(got["out"][1], 0)
        assert np.isneginf(got["lse"][1]).all()
        for d in dev:
            d.free()


def test_a_cache_past_32_bit_offsets(gpu_ctx):
    """Pages whose bytes lie behind 2^32."""
    rng, page, pages = np.random.default_rng(13), 1024, 15000
    with open_cache(gpu_ctx, "576", pages, page, 1, 32) as cache:       # 15.4 M tokens of 288 bytes
        table = np.array([[14999, 3, 14990]], np.int32)
        lengths = np.array([2500])
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round(rng.standard_normal((1, 32, 576)).astype(np.float32))
        want = oracle.attend(q, keys, values, lengths, [1], 0.1)
        check(cache.attend(bf16_bits(q), table, lengths, 0.1), q, keys, lengths, 0.1, *want)


@pytest.mark.parametrize("kind,heads,kv_heads,counts", [("512", 64, 1, [1, 1, 1]), ("128", 32, 8, [40, 1, 300]), ("576", 16, 1, [2, 2, 2])])
def test_captured_attention_follows_the_lengths(gpu_ctx, kind, heads, kv_heads, counts):
    """One captured step, replayed as the sequences grow; every replay equals the eager call, and a second graph over the
    same workspace does not disturb the first."""
    rng, page, counts = np.random.default_rng(14), 16, np.array(counts)
    most = np.array([2000, 500, 700])
    table, pages = pages_for(rng, most, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        fill(cache, rng, table, most)
        t = int(counts.sum())
        first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        q = bf16_bits(rng.standard_normal((t, heads, cache.width)).astype(np.float32))
        out0 = np.full((t, heads, cache.value_width), 7, np.uint16)
        dev = [gpu_ctx.upload(a) for a in (q, table, most.astype(np.int32), first, out0, out0)]
        stream = gpu_ctx.stream()
        graphs = [Graph(gpu_ctx, stream, lambda d=d: cache.attend_device(dev[0], t, dev[1], table.shape[1], dev[2], 3, d, 0.1, dev[3], stream=stream))
                  for d in dev[4:]]
        for lengths in ([2000, 500, 700], [40, 1, 300], [1999, 17, 699], [1, 0, 5]):
            dev[2].upload(np.array(lengths, np.int32))
            gpu_ctx.sync()
            eager = cache.attend(q, table, np.array(lengths), 0.1, counts)["out"]
            for g in (0, 1, 0):
                dev[4 + g].upload(out0)
                gpu_ctx.sync()
                graphs[g].launch()
                np.testing.assert_array_equal(dev[4 + g].download(), eager)
        for g in graphs:
            g.close()
        gpu_ctx.destroy_stream(stream)
        for d in dev:
            d.free()


def test_host_calls_refuse(gpu_ctx):
    cache = open_cache(gpu_ctx, "64", 4, 16, 2, 4, max_tokens=8, max_batch=2)
    k, slots = np.zeros((3, 2, 64), np.float32), np.arange(3)
    for args in ((k[0], slots, k), (k, slots, None), (k, slots[:2], k), (k, slots + 62, k), (k, np.array([1, 1, 2]), k), (k, slots * 1.0, k),
                 (k, slots, bf16_bits(k)), (k, slots, k[:2]), (k.astype(np.float64), slots, k), (k, slots, k, None, slots)):
        with pytest.raises(ValueError):
            cache.append(*args)
    q, table, lengths = np.zeros((2, 4, 64), np.uint16), np.zeros((2, 2), np.int32), np.array([3, 32])
    for args in ((q.astype(np.float32), table, lengths, 1.0), (q[:1], table, lengths, 1.0), (q, table[0], lengths, 1.0), (q, table[:1], lengths, 1.0),
                 (q, table, lengths + 1, 1.0), (q, table, lengths - 4, 1.0), (q, table + 4, lengths, 1.0), (q, table - 1, lengths, 1.0),
                 (q, table * 1.0, lengths, 1.0), (q, table, lengths, 0.0), (q, table, lengths, 1.0, [1, 2]), (q, table, lengths, 1.0, [-1, 2]),
                 (q, table, lengths, 1.0, None, -1), (q, table, lengths, 1.0, None, 0, np.zeros(3)), (np.zeros((10, 4, 64), np.uint16), table, lengths, 1.0)):
        with pytest.raises(ValueError):
            cache.attend(*args)
    with pytest.raises(ValueError):
        cache.read([4])
    assert cache.attend(q[:0], table[:0], lengths[:0], 1.0)["out"].shape == (0, 4, 64)
    cache.close()
    for call in (lambda: cache.read([0]), lambda: cache.append(k, slots, k), lambda: cache.attend(q, table, lengths, 1.0)):
        with pytest.raises(RuntimeError):
            call()
