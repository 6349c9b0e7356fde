"""Logits far from zero, up to 2^120 and down to -2^120: the largest ones share the row, and nothing overflows.

One column of the keys is 1, 2, 3 or 4, and the query is zero elsewhere, so logits are multiples of one number that is at least
2^8: only the tokens of the largest have a share above e^-256, each the same. Their powers 2^(c s - m) are not 1, and differ
between steps and workgroups, whose maxima m are products rounded to FP32 and raised by whole numbers. Each power is rounded to
BF16 for the products (2^-8 of it) while the sum takes it as it is, so the mean of their values v is off by 2^-8 of the mean of
|v|; some hundred additions in FP32 change it by 2^-12 of that. The result is rounded to BF16 once more."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_values
from tests.test_gpu_kv4 import open_cache, pages_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("512", 16, 1), ("576", 40, 1), ("64", 14, 2), ("128", 32, 8), ("256", 8, 2)])
@pytest.mark.parametrize("power", [8, 20, 23, 24, 28, 30, 33, 60, 118])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_logits_share_the_row(gpu_ctx, kind, heads, kv_heads, power, sign):
    rng, page = np.random.default_rng(power), 64
    lengths = np.array([1, 40, 700, 9000])
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        total = int(lengths.sum())
        grid = np.concatenate([oracle.GRID, -oracle.GRID[1:]])
        k, v = (rng.choice(grid, (total, kv_heads, w)).astype(np.float32) for w in (cache.width, cache.value_width))
        k[..., ::32] = 6                 # one scale for every block
        v[..., ::32] = 6
        k[..., 5] = rng.choice([1, 2, 3, 4], (total, kv_heads), p=[.05, .45, .45, .05])
        slots = np.concatenate([table[b][np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page for b, n in enumerate(lengths)])
        cache.append(k, slots, v if cache.apart else None)
        q = np.zeros((4, heads, cache.width), np.float32)
        q[..., 5] = sign * 2.0 ** min(power, 60)
        got = cache.attend(bf16_bits(q), table, lengths, 2.0 ** (power - min(power, 60)))
        first = np.concatenate([[0], np.cumsum(lengths)])
        for b in range(4):
            part = slice(first[b], first[b + 1])
            for h in range(heads):
                j = h // (heads // kv_heads)
                logit = sign * k[part, j, 5].astype(np.float64)
                best = logit == logit.max()
                tied = (v if cache.apart else k[..., :cache.value_width])[part, j][best].astype(np.float64)
                want, limit = tied.mean(0), 2.0 ** -8 * (1 + 2.0 ** -4) * np.abs(tied).mean(0)
                error = np.abs(bf16_values(got["out"][b, h]) - want)
                worst = np.max(error - limit - 2.0 ** -8 * (np.abs(want) + limit))
                assert worst <= 0, (b, h, worst)
                lse = logit.max() * 2.0 ** power + np.log(best.sum())
                assert abs(got["lse"][b, h] - lse) <= 2.0 ** -21 * abs(lse), (b, h, got["lse"][b, h], lse)
