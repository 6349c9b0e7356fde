"""Attention's ways of dividing rows: how many rows a workgroup takes at once follows from what the tables can hold, so wide
tables take short sequences through the kernels of long ones. Tolerances as for the narrow tables."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_round, bf16_values
from tests.test_gpu_kv4 import ATTENDS, check, fill, open_cache, pages_for

pytestmark = pytest.mark.gpu


def columns_for(steps, kind, kv_heads, rows, batch, page, least):
    """The columns at which a wave would have `steps` steps of 32 rows and 32 tokens if the tables were full."""
    workgroups = 256 * {"64": 3, "128": 2}.get(kind, 1)
    tokens = 32 * 4 * workgroups * steps / (batch * kv_heads * -(-rows // 32))
    return min(max(int(tokens) // page, least), 2 ** 30 // page, 1 << 19)


@pytest.mark.parametrize("steps", [40, 1000])
@pytest.mark.parametrize("kind,heads,kv_heads,lengths,counts,page,window,sinks", [a for a in ATTENDS if not a[6]])
def test_attend_over_wide_tables(gpu_ctx, kind, heads, kv_heads, lengths, counts, page, window, sinks, steps):
    rng = np.random.default_rng(heads + sum(lengths) + steps)
    lengths = np.array(lengths)
    n = np.ones(len(lengths), int) if counts is None else np.array(counts)
    rows = -(-int(n.sum()) // len(n)) * (heads // kv_heads)
    least = max(int(-(-lengths // page).max()), 1)
    table, pages = pages_for(rng, lengths, page, columns=columns_for(steps, kind, kv_heads, rows, len(n), page, least))
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round((rng.standard_normal((int(n.sum()), heads, cache.width)) * 2).astype(np.float32))
        s = (rng.standard_normal(heads) * 2).astype(np.float32) if sinks else None
        scale = cache.width ** -0.5
        want = oracle.attend(q, keys, values, lengths, n, scale, 0, s)
        check(cache.attend(bf16_bits(q), table, lengths, scale, counts, 0, s), q, keys, lengths, scale, *want)


@pytest.mark.parametrize("kind,heads,kv_heads,counts", [("512", 64, 1, [300, 20]), ("576", 16, 1, [400, 9]), ("64", 14, 2, [250, 9]),
                                                        ("128", 32, 8, [300, 70]), ("256", 8, 2, [129, 33])])
@pytest.mark.parametrize("window", [1, 40, 128])
@pytest.mark.parametrize("columns", [None, 1 << 16])
def test_windows_of_prompts(gpu_ctx, kind, heads, kv_heads, counts, window, columns):
    """Every row tile begins elsewhere, and most of the cache is seen by nobody."""
    rng, page = np.random.default_rng(window), 16
    counts = np.array(counts)
    lengths = counts + [100, 3]
    table, pages = pages_for(rng, lengths, page, columns=columns)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round(rng.standard_normal((int(counts.sum()), heads, cache.width)).astype(np.float32))
        scale = cache.width ** -0.5
        want = oracle.attend(q, keys, values, lengths, counts, scale, window)
        check(cache.attend(bf16_bits(q), table, lengths, scale, counts, window), q, keys, lengths, scale, *want)


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 40, 1), ("576", 128, 1), ("64", 14, 2), ("128", 32, 8), ("256", 8, 2)])
@pytest.mark.parametrize("columns", [None, 1 << 14])
def test_more_units_than_a_workgroup_counts(gpu_ctx, kind, heads, kv_heads, columns):
    """Past 1024 row tiles the plan is made by a kernel of its own, by what the call could hold; empty sequences between."""
    rng, page = np.random.default_rng(heads), 16
    lengths = np.concatenate([rng.integers(0, 40, 1100), [3000]])
    lengths[::7] = 0
    counts = (lengths > 0).astype(int)
    table, pages = pages_for(rng, lengths, page, columns=columns and max(columns, 188))
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads, max_batch=2048) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round(rng.standard_normal((int(counts.sum()), heads, cache.width)).astype(np.float32))
        want = oracle.attend(q, keys, values, lengths, counts, 0.05)
        check(cache.attend(bf16_bits(q), table, lengths, 0.05, counts), q, keys, lengths, 0.05, *want)


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("576", 128, 1), ("64", 14, 2), ("128", 32, 8), ("256", 8, 2)])
@pytest.mark.parametrize("columns", [1, 1 << 18])
def test_one_token_is_its_values(gpu_ctx, kind, heads, kv_heads, columns):
    """Its probability is 1 to 2^-20 whatever its logit, and a value has two significant bits: nothing is left to round."""
    rng = np.random.default_rng(heads)
    lengths = np.ones(9, int)
    table, pages = pages_for(rng, lengths, 16, columns=columns)
    with open_cache(gpu_ctx, kind, pages, 16, kv_heads, heads) as cache:
        _, values = fill(cache, rng, table, lengths)
        q = bf16_round((rng.standard_normal((9, heads, cache.width)) * np.exp2(np.arange(9) - 6)[:, None, None]).astype(np.float32))
        got = bf16_values(cache.attend(bf16_bits(q), table, lengths, cache.width ** -0.5)["out"])
        for b in range(9):
            np.testing.assert_array_equal(got[b], values[b][0].repeat(heads // kv_heads, 0))


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 40, 1), ("576", 16, 1), ("64", 14, 2), ("128", 32, 8), ("256", 8, 2)])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("columns", [None, 1 << 14])
def test_some_hundred_sequences(gpu_ctx, kind, heads, kv_heads, given, columns):
    """More row tiles than a wave has lanes, fewer than a workgroup counts, with and without rows of empty sequences."""
    rng, page = np.random.default_rng(heads + given), 16
    lengths = np.concatenate([rng.integers(0, 90, 180), [2000, 0, 1]])
    counts = (rng.integers(0, 3, lengths.size) * (lengths > 2)) if given else np.ones(lengths.size, int)
    table, pages = pages_for(rng, lengths, page, columns=columns)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        keys, values = fill(cache, rng, table, lengths)
        q = bf16_round(rng.standard_normal((int(counts.sum()), heads, cache.width)).astype(np.float32))
        want = oracle.attend(q, keys, values, lengths, counts, 0.05)
        check(cache.attend(bf16_bits(q), table, lengths, 0.05, counts if given else None), q, keys, lengths, 0.05, *want)
