"""Attention where single channels of the queries or keys are far larger than their neighbours.

Of eight neighbouring products (columns 8 i to 8 i + 7) the matrix units cut each but the largest towards zero at 2^-13 of the
power of two of its factors, which is at most twice 2^-13 of the largest product (twice where a code of 0.5 has a part in it):
seven of them lose 2^-12 of it each at most. That happens for the first term of the query and for the second, whose products are
at most 2^-4 of the first's: 7 (1 + 2^-4 + 2^-4) 2^-12 <= 2^-9 of the sum of the eights' largest products. The two terms hold a
query's value to 2^-21 of the largest of its block of 32: the block's largest is in [2^7, 2^8) units of the first term's scale, and
the second's smallest step is 2^-9 2^-4 of a unit, half of which is 2^-14 units. Beside that a logit is a chain of additions and roundings as on any values, 56 2^-24 of the sum of its products' magnitudes. A logit that is off by d
changes each probability's share by a factor of at most e^(2 d); probabilities and results are rounded to BF16, 2^-8 each."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_round, bf16_values
from tests.test_gpu_kv4 import open_cache, pages_for

pytestmark = pytest.mark.gpu
HEADS = {"64": (14, 2), "128": (32, 8), "256": (8, 2), "512": (64, 1), "576": (16, 1)}


def logit_error(q, k, scale):
    """[rows, tokens] of q [rows, width] and k [tokens, width], both float64."""
    products = np.abs(q[:, None] * k[None])
    largest = products.reshape(*products.shape[:2], -1, 8).max(-1).sum(-1)
    blocks = lambda a: np.abs(a).reshape(a.shape[0], -1, 32)  # noqa: E731
    held = blocks(q).max(-1) @ blocks(k).sum(-1).T
    return (2.0 ** -9 * largest + 2.0 ** -21 * held + 56 * 2.0 ** -24 * products.sum(-1)) * scale + 2.0 ** -22


def lifted(rng, shape, how, lift):
    """Normal values; "eights": one of every eight lift times as large, "channel": the same one column of all."""
    x = rng.standard_normal(shape)
    columns = np.arange(0, shape[-1], 8) + rng.integers(0, 8, shape[-1] // 8) if how == "eights" else [shape[-1] // 2 + 3]
    if how != "plain":
        x[..., columns] *= lift
    return bf16_round(x.astype(np.float32))


@pytest.mark.parametrize("kind", HEADS)
@pytest.mark.parametrize("q_how,k_how", [("eights", "plain"), ("channel", "plain"), ("eights", "channel"), ("channel", "channel"), ("plain", "eights")])
@pytest.mark.parametrize("lift", [8, 30, 100, 1000, 1e5])
def test_channels_larger_than_their_neighbours(gpu_ctx, kind, q_how, k_how, lift):
    rng = np.random.default_rng(int(lift) + int(kind))
    heads, kv_heads = HEADS[kind]
    group, page, lengths = heads // kv_heads, 16, np.array([1, 90, 33])
    table, pages = pages_for(rng, lengths, page)
    with open_cache(gpu_ctx, kind, pages, page, kv_heads, heads) as cache:
        k = lifted(rng, (int(lengths.sum()), kv_heads, cache.width), k_how, lift)
        v = lifted(rng, (int(lengths.sum()), kv_heads, cache.width), "plain", 1) if cache.apart else None
        slots = np.concatenate([table[b][np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page for b, n in enumerate(lengths)])
        cache.append(k, slots, v)
        q = lifted(rng, (3, heads, cache.width), q_how, lift)
        kd = oracle.decode(*oracle.encode(k))
        vd = kd[..., :cache.value_width] if v is None else oracle.decode(*oracle.encode(v))
        first = np.concatenate([[0], np.cumsum(lengths)])
        keys, values = ([a[first[b]:first[b + 1]] for b in range(3)] for a in (kd, vd))
        top = max(np.abs(np.einsum("hd,tjd->htj", q[b].astype(np.float64), keys[b])).max() for b in range(3))
        for scale in (float(np.float32(min(cache.width ** -0.5, 8 / top))), cache.width ** -0.5):
            want, lse, size = oracle.attend(q, keys, values, lengths, [1] * 3, scale)
            got = cache.attend(bf16_bits(q), table, lengths, scale)
            for b in range(3):
                for j in range(kv_heads):
                    rows = slice(j * group, (j + 1) * group)
                    d = logit_error(q[b, rows].astype(np.float64), keys[b][:, j], scale).max(1)
                    error = np.abs(got["lse"][b, rows].astype(np.float64) - lse[b, rows])
                    assert np.all(error <= d + 2.0 ** -22 * (1 + np.abs(lse[b, rows])) + 64 * 2.0 ** -24)
                    change = np.expm1(2 * np.minimum(d, 300))[:, None]
                    limit = (change + 2.0 ** -8 * (1 + 2.0 ** -8) * (1 + change)) * size[b, rows] + 1e-30
                    limit = limit + 2.0 ** -8 * (np.abs(want[b, rows]) + limit)
                    assert np.all(np.abs(bf16_values(got["out"][b, rows]) - want[b, rows]) <= limit)
