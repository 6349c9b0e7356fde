"""Weights that are not finite (load refuses them, load_device cannot see them) stay with the requests that name their
slot, and leave with it: a smaller adapter loaded over them shows nothing of what lies past its ranks."""

import numpy as np
import pytest

from oracle import adapters as oracle
from oracle.formats import bf16_bits, bf16_values
from vesper_amd.adapters import AdapterBank

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [3, 40, 100, 200])
@pytest.mark.parametrize("max_rank,width", [(16, 264), (32, 264), (64, 1544), (128, 520), (200, 1544)])
def test_spoiled_weights_stay_with_their_slot(gpu_ctx, tokens, max_rank, width):
    rng = np.random.default_rng(tokens + max_rank)
    rows = 72

    def small(rank):
        return [bf16_bits(rng.integers(-2, 3, s).astype(np.float32)) for s in ((rank, width), (rows, rank))]
    x = bf16_bits(rng.integers(-2, 3, (tokens, width)).astype(np.float32))
    base = rng.integers(-99, 100, (tokens, rows)).astype(np.float32)
    ids = (np.arange(tokens) % 3 - 1).astype(np.int32)   # none, slot 0, slot 1
    spoiled = [np.where(rng.random(a.shape) < 0.5, np.uint16(0x7F80), np.uint16(0x7FC0)) for a in small(max_rank)]
    with AdapterBank(gpu_ctx, rows, width, 2, max_rank, tokens) as bank:
        dev = [gpu_ctx.upload(a) for a in spoiled]
        bank.load_device(0, *dev, max_rank)
        good = small(max_rank - 3)
        bank.load(1, *good, -2.0)
        adapters = {1: (*map(bf16_values, good), -2.0)}
        want = bf16_bits(oracle.apply(bf16_values(x), ids, base, adapters)[0].astype(np.float32))
        got = bank.apply(x, ids, base)
        np.testing.assert_array_equal(got[ids != 0], want[ids != 0])
        assert np.isnan(bf16_values(got[ids == 0])).all()
        rank = max(1, max_rank // 3)
        smaller = small(rank)
        bank.load(0, *smaller, 0.5)
        adapters[0] = (*map(bf16_values, smaller), 0.5)
        want = bf16_bits(oracle.apply(bf16_values(x), ids, base, adapters)[0].astype(np.float32))
        np.testing.assert_array_equal(bank.apply(x, ids, base), want)
        for a in dev:
            a.free()
