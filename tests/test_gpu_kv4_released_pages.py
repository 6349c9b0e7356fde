"""Windows: pages that no row sees any more may have left the table, and come to other sequences; results are those of the whole
table, bit for bit. A page that one row still sees may not."""

import numpy as np
import pytest

from oracle.formats import bf16_bits, bf16_round
from tests.test_gpu_kv4 import fill, open_cache, pages_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,heads,kv_heads", [("512", 64, 1), ("576", 16, 1), ("64", 14, 2), ("128", 32, 8), ("256", 8, 2)])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 40, 1000])
@pytest.mark.parametrize("given", [False, True])
def test_pages_before_the_windows(gpu_ctx, kind, heads, kv_heads, window, given):
    rng, page = np.random.default_rng(window), 16
    lengths = np.array([200, 33, 16, 0, 700, 97])
    counts = np.array([1, 5, 2, 0, 40, 0]) if given else np.ones(6, int)
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        fill(cache, rng, table, lengths)
        q = bf16_bits(bf16_round(rng.standard_normal((int(counts.sum()), heads, cache.width)).astype(np.float32)))
        args = (lengths, 0.1, counts if given else None, window)
        want = cache.attend(q, table, *args)
        seen = np.maximum(lengths - counts + 1 - window, 0) // page          # the first page that a row sees
        released = np.arange(table.shape[1]) < seen[:, None]
        for other in (-1, pages, table[4, 0]):                               # nobody's, no page at all, another sequence's
            got = cache.attend(q, np.where(released, other, table), *args)
            for name in want:
                np.testing.assert_array_equal(got[name], want[name])
        if (seen > 0).any():
            one = table.copy()
            b = int(np.argmax(seen))
            one[b, seen[b]] = -1
            with pytest.raises(ValueError):
                cache.attend(q, one, *args)
            with pytest.raises(ValueError):
                cache.attend(q, np.where(released, -1, table), *args[:3])
