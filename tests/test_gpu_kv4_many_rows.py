"""An append of the most tokens: 2^27 rows of keys and values on 32 lanes each, 2^32 lanes in all, which no launch can have. Few of
the tokens have slots; their codes, positions and rounded values are those of a small call."""

import numpy as np
import pytest

from oracle.formats import bf16_bits
from tests.test_gpu_kv4 import open_cache
from vesper_amd.attention import HeadRotation, rotation_table

pytestmark = pytest.mark.gpu


def test_the_most_tokens(gpu_ctx):
    rng, tokens, heads, width = np.random.default_rng(0), 1 << 20, 64, 256
    at = np.array([0, 7, 32767, 65535, 65536, 1 << 19, (1 << 20) - 2, (1 << 20) - 1])
    rows = bf16_bits(rng.standard_normal((len(at), heads, width)).astype(np.float32))
    slots = np.full(tokens, -1, np.int64)
    slots[at] = rng.permutation(16)[:len(at)]
    positions = np.full(tokens, -1, np.int32)
    positions[at] = rng.integers(0, 50, len(at))
    with open_cache(gpu_ctx, "256", 1, 16, heads, heads) as cache, open_cache(gpu_ctx, "256", 1, 16, heads, heads) as small, \
            HeadRotation(gpu_ctx, width, width, 64, table=rotation_table(50, 64)) as rot:
        for d in cache._owned[:4] + small._owned[:4]:
            d.upload(np.zeros(d.shape, np.uint8))
        rounded = small.append(rows, slots[at], rows, rot, positions[at])
        step = heads * width * 2
        x, y = gpu_ctx.malloc(tokens * step), gpu_ctx.malloc(tokens * step)     # 34 GB each, of which nothing else is looked at
        try:
            for t, row in zip(at, rows):
                gpu_ctx.copy_h2d(x + int(t) * step, row)
            dev = [gpu_ctx.upload(a) for a in (slots, positions)]
            for name in "kv":
                to = {f"{name}_rounded_ptr": y}
                cache.append_device(x, dev[0], tokens, x, rot, dev[1], **to)
                gpu_ctx.sync()
                for i, t in enumerate(at):
                    np.testing.assert_array_equal(gpu_ctx.download(y + int(t) * step, (heads, width), np.uint16), rounded[name][i])
            for d in dev:
                d.free()
        finally:
            gpu_ctx.free(x)
            gpu_ctx.free(y)
        want, got = small.read([0]), cache.read([0])
        for name in want:
            np.testing.assert_array_equal(got[name], want[name])
        assert want["v_codes"].any()
