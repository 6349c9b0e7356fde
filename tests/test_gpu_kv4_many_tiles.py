"""More row tiles than a workgroup counts, so that a kernel of its own makes the plan, for every number of rows that a tile can
have: sequences of several steps each, whole and in parts, with one row or several, some with none. Some sequences are compared
with the 64-bit oracle, all of them with calls of fewer, whose workgroups count for themselves: two results are each within the
oracle's limit, at most (2^-7 + 2^-8) of the largest value here, where logits are off by less than 2^-10, so within 2^-5 of each other, and
their logarithms of sums within 2^-9."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_round, bf16_values
from tests.test_gpu_kv4 import check, fill, open_cache

pytestmark = pytest.mark.gpu


# heads of a key head that leave tiles of 32 rows (latents, values apart), 64 and 128
@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 8, 1), ("576", 16, 1), ("512", 32, 1), ("512", 4, 2), ("576", 40, 1), ("64", 4, 2),
                                                ("128", 8, 1), ("256", 2, 1), ("128", 40, 1), ("64", 80, 1)])
@pytest.mark.parametrize("longest,columns", [(70, None), (250, 1 << 13)])
@pytest.mark.parametrize("given", [False, True])
def test_plans_of_many_tiles(gpu_ctx, kind, heads, kv_heads, longest, columns, given):
    rng, page, batch = np.random.default_rng(heads + longest + given), 16, 1030
    lengths = rng.integers(0, longest + 1, batch)
    lengths[5], lengths[700] = 0, 3 * longest
    counts = rng.integers(0, 3, batch) if given else np.ones(batch, int)
    counts[700] = 1
    first = np.concatenate([[0], np.cumsum(counts)])
    pages = 60                                               # which the sequences share, each in an order of its own
    table = rng.integers(0, pages, (batch, columns or -(-int(lengths.max()) // page))).astype(np.int32)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads, max_batch=2048) as cache:
        (k,), (v,) = fill(cache, rng, np.arange(pages)[None], np.array([pages * page]))
        at = [(table[b][np.arange(n) // page] * page + np.arange(n) % page) for b, n in enumerate(lengths)]
        keys, values = [k[a] for a in at], [v[a] for a in at]
        q = bf16_round((rng.standard_normal((int(counts.sum()), heads, cache.width)) * 2).astype(np.float32))
        scale = cache.width ** -0.5
        got = cache.attend(bf16_bits(q), table, lengths, scale, counts if given else None)
        top = np.abs(v).max()
        for b in range(0, batch, 103):
            part = slice(b, b + 103)
            few = cache.attend(bf16_bits(q[first[b]:first[b + 103]]), table[part], lengths[part], scale, counts[part] if given else None)
            one = {k: a[first[b]:first[b + 103]] for k, a in got.items()}
            np.testing.assert_array_equal(np.isneginf(one["lse"]), np.isneginf(few["lse"]))
            live = ~np.isneginf(few["lse"])
            np.testing.assert_allclose(one["lse"][live], few["lse"][live], rtol=0, atol=2.0 ** -9)
            np.testing.assert_allclose(bf16_values(one["out"]), bf16_values(few["out"]), rtol=0, atol=2.0 ** -5 * top)
        some = heads // kv_heads * np.arange(kv_heads)        # the oracle on one head of each key head
        for b in [0, 5, 700, batch - 1, *rng.integers(0, batch, 20)]:
            rows = slice(first[b], first[b + 1])
            want = oracle.attend(q[rows][:, some], keys[b:b + 1], values[b:b + 1], lengths[b:b + 1], counts[b:b + 1], scale)
            if counts[b] and lengths[b]:
                check({k: a[rows][:, some] for k, a in got.items()}, q[rows][:, some], keys[b:b + 1], lengths[b:b + 1], scale, *want)
