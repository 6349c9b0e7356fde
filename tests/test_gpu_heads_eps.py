"""Gradients of heads with eps = 0: rows that are no token, and the lanes behind the last row, have no root; they get zeros
and add nothing, also where a weight is not finite. Tolerances as in test_gpu_heads.py."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_values
from vesper_amd.attention import HeadRotation, rotation_table

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rows(rng, shape, dtype):
    x = rng.standard_normal(shape).astype(np.float32)
    return bf16_bits(x) if dtype == "bf16" else x


def values(a):
    return bf16_values(a).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


# tokens x heads leave a remainder of the rows that a workgroup takes at once (32, 16, 8 and 4), and less than one of them
@pytest.mark.parametrize("tokens,heads,width", [(1, 1, 64), (3, 1, 64), (37, 1, 64), (5, 3, 128), (70, 3, 128), (9, 1, 256), (1, 3, 512), (3, 3, 512),
                                                (5, 1, 1024), (3, 1, 4096), (900, 7, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("padded", [False, True])
def test_gradients_without_eps(gpu_ctx, tokens, heads, width, dtype, padded):
    rng = np.random.default_rng(tokens * width + heads)
    x, dy = rows(rng, (tokens, heads, width), dtype), rows(rng, (tokens, heads, width), dtype)
    table, positions = rotation_table(20, 16), rng.integers(0, 20, tokens)
    if padded:
        positions[::3] = -1
    live = positions >= 0
    weight = rng.uniform(0.5, 1.5, width).astype(np.float32)
    with HeadRotation(gpu_ctx, width, width, 16, eps=0.0, table=table) as rot:
        got = rot.backward(dy, x, positions, weight)
    args = dict(norm=width, weight=weight, first=width - 16, dims=16, eps=0.0)
    xl, dyl = values(x)[live], values(dy)[live]
    dx, dw = oracle.heads_backward(dyl, xl, table, positions[live], **args)
    np.testing.assert_array_equal(values(got["dx"])[~live], 0)
    r = 1 / np.sqrt(np.mean(xl ** 2, -1, keepdims=True))
    u, size = np.abs(xl * r), np.abs(dyl)
    size[..., width - 16:] = (size[..., width - 16::2] + size[..., width - 15::2]).repeat(2, -1)   # |a| + |b| of a turned pair
    gw = size * weight
    limit = r * U * (16 * gw + 96 * u * np.mean(gw * u, -1, keepdims=True)) + 1e-37
    if dtype == "bf16":
        limit = limit + 2.0 ** -8 * (np.abs(dx) + limit)
    assert np.all(np.abs(values(got["dx"])[live] - dx) <= limit)
    assert np.all(np.abs(got["dweight"] - dw) <= (tokens * heads / 512 + 100) * U * np.sum(size * u, (0, 1)) + 1e-37)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_rows_of_no_token_are_zero_beside_weights_that_are_not_finite(gpu_ctx, eps):
    rng = np.random.default_rng(1)
    x, dy = rows(rng, (6, 2, 128), "f32"), rows(rng, (6, 2, 128), "f32")
    x[1], dy[4] = np.nan, np.inf
    weight = np.ones(128, np.float32)
    weight[3], weight[70] = np.inf, np.nan
    positions = np.array([2, -1, 0, -1, -1, 7])
    with HeadRotation(gpu_ctx, 128, 128, 16, eps=eps, table=rotation_table(8, 16)) as rot:
        got = rot.backward(dy, x, positions, weight)
    np.testing.assert_array_equal(got["dx"][positions < 0], 0)
    assert np.isfinite(got["dweight"]).all()     # the weights' gradient does not depend on them
