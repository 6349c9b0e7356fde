"""Windows of more positions than a sequence has, up to past 32 bits, are none."""

import numpy as np
import pytest

from oracle.formats import bf16_bits, bf16_round
from tests.test_gpu_kv4 import fill, open_cache, pages_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("576", 16, 1), ("64", 4, 4), ("128", 32, 8), ("256", 8, 2)])
def test_windows_past_the_sequences(gpu_ctx, kind, heads, kv_heads):
    rng, page = np.random.default_rng(heads), 16
    lengths, counts = np.array([100, 1, 700]), np.array([5, 1, 40])
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        fill(cache, rng, table, lengths)
        q = bf16_bits(bf16_round(rng.standard_normal((46, heads, cache.width)).astype(np.float32)))
        want = cache.attend(q, table, lengths, 0.1, counts)
        for window in (700, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5):
            got = cache.attend(q, table, lengths, 0.1, counts, window)
            for name in want:
                np.testing.assert_array_equal(got[name], want[name])
