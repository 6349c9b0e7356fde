"""Adapters of calls whose plan is made in three launches, up to the most tokens: small integers, exact."""

import numpy as np
import pytest

from tests.test_gpu_adapters_wide import fill, make, run
from vesper_amd.adapters import AdapterBank

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,slots,rank", [(49152, 3, 16), (49153, 3, 16), (16400, 1024, 8), (100003, 40, 64),
                                               (1 << 18, 1024, 16), (1 << 18, 2, 136)])
def test_many_tokens(gpu_ctx, tokens, slots, rank):
    rng = np.random.default_rng(tokens + slots)
    rows, width = 16, 24
    with AdapterBank(gpu_ctx, rows, width, slots, rank, tokens) as bank:
        adapters = fill(gpu_ctx, bank, [make(rng, rows, width, r) for r in (rank, rank // 2)], (1.0, -2.0, 0.5), slots - 1)
        run(gpu_ctx, bank, rng.integers(-1, slots, tokens), adapters, rank, "f32", (False, True))
