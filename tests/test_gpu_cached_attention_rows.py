"""Rows of a step that no sequence has: their y is zero, whatever the steps before left in the layer's buffers."""

import numpy as np
import pytest

from oracle.formats import bf16_bits
from tests.test_gpu_cached_attention import PAGE, TABLE, options, projections  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_rows_behind_the_last_sequence_are_zero(projections):  # noqa: F811
    rng = np.random.default_rng(5)
    table, lengths = np.array([[0], [1]], np.int32), np.array([3, 2])
    x = bf16_bits(rng.standard_normal((7, 5120)).astype(np.float32))
    positions, slots = np.array([0, 1, 2, 0, 1, -1, 4]), np.array([0, 1, 2, PAGE, PAGE + 1, -1, 2 * PAGE])
    with projections.open_cache(3, PAGE, TABLE, **options(rng, max_tokens=7)) as layer:
        got = []
        for _ in range(2):
            other = bf16_bits((rng.standard_normal((7, 5120)) * 3).astype(np.float32))
            at = np.arange(7)
            layer.step(other, at, at + 2 * PAGE, np.array([[2]], np.int32), np.array([7]), [7])   # another session's step
            got.append(layer.step(x, positions, slots, table, lengths, [3, 2]))
        np.testing.assert_array_equal(got[0], got[1])
        np.testing.assert_array_equal(got[0][5:], 0)
        assert np.any(got[0][:5], -1).all()
        # their latents are stored where they have a slot
        stored = layer.cache.read([2])["k_codes"][0, 0, 0]
        layer.step(x[6:], positions[6:], np.array([0]), table[:1], np.array([5]))
        np.testing.assert_array_equal(stored, layer.cache.read([0])["k_codes"][0, 0, 0])
        np.testing.assert_array_equal(layer.step(x, positions, slots, table, np.zeros(2, int), [0, 0]), 0)
