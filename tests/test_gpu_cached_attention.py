"""An attention layer over its cache: from the layer's input to its output, as a decode or prompt step runs it.

The step is its parts called one by one, bit for bit, and its attention is the 64-bit oracle's over what the cache holds: a
probability and the result are rounded to BF16 once each (2^-8 relative each at most), the rotation back adds the errors of
two values and one rounding more."""

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_values
from oracle.projections import fp8_weights
from tests.test_gpu_scratch import Graph
from vesper_amd.attention import HeadRotation, rotation_table
from vesper_amd.projections import FP8_LAYOUT, WO_A, NativeProjections

pytestmark = pytest.mark.gpu
HEADS, WIDTH, DIMS, PAGE = 64, 512, 64, 16
TABLE = rotation_table(600, DIMS)


@pytest.fixture(scope="module")
def projections():
    rng = np.random.default_rng(3)
    arrays = {}
    for name, (rows, width) in dict(FP8_LAYOUT, wo_a=WO_A).items():
        w, s = fp8_weights(rng, rows, width, 32)
        arrays[f"layers.0.attn.{name}.weight"], arrays[f"layers.0.attn.{name}.scale"] = w, s
    with NativeProjections(arrays) as proj:
        yield proj


def options(rng, **more):
    return dict(dict(max_tokens=80, max_batch=4, q_norm=(rng.random(1280) + 0.5).astype(np.float32),
                     kv_norm=(rng.random(WIDTH) + 0.5).astype(np.float32), sinks=rng.standard_normal(HEADS).astype(np.float32)), **more)


def one_by_one(proj, layer, opened, x, positions, slots, table, lengths, counts):
    """The same through the parts' own calls, over layer's cache as the step has left it."""
    t = x.shape[0]
    with HeadRotation(proj.ctx, 1280, norm=1280) as down:
        qa = down.apply(proj.fp8("wq_a", x)["output_bf16"].reshape(t, 1, 1280), weight=opened["q_norm"]).reshape(t, 1280)
    q = layer.heads.apply(proj.fp8("wq_b", qa)["output_bf16"].reshape(t, HEADS, WIDTH), positions)
    k = layer.heads.apply(proj.fp8("wkv", x)["output_bf16"].reshape(t, 1, WIDTH), positions, opened["kv_norm"])
    got = layer.cache.attend(q, table, lengths, layer.scale, counts, layer.window, opened["sinks"])
    back = layer.back.apply(got["out"], positions, inverse=True)
    y = np.concatenate([proj.grouped(np.ascontiguousarray(back[i:i + 32]).reshape(-1, 8, 4096))["output_bf16"] for i in range(0, t, 32)])
    return q, k, back, proj.fp8("wo_b", np.ascontiguousarray(y.reshape(t, -1)))["output_bf16"]


def slots_of(table, positions):
    return np.concatenate([table[b][p // PAGE].astype(np.int64) * PAGE + p % PAGE for b, p in enumerate(positions)])


@pytest.mark.parametrize("window", [0, 24])
def test_steps_are_their_parts_and_the_oracle(projections, window):
    """A prompt of three sequences, then a draft of several tokens, then single tokens."""
    rng = np.random.default_rng(window)
    table = rng.permutation(3 * 6).astype(np.int32).reshape(3, 6)
    opened = options(rng, window=window)
    layer = projections.open_cache(18, PAGE, TABLE, **opened)
    lengths = np.zeros(3, np.int64)
    cached = [np.zeros((0, WIDTH)) for _ in range(3)]
    for counts in ([40, 7, 23], [3, 0, 4], [1, 1, 1]):
        positions = [np.arange(lengths[b], lengths[b] + n) for b, n in enumerate(counts)]
        lengths = lengths + counts
        flat = np.concatenate(positions)
        x = bf16_bits(rng.standard_normal((sum(counts), 5120)).astype(np.float32))
        slots = slots_of(table, positions)
        y = layer.step(x, flat, slots, table, lengths, counts if len(set(counts)) > 1 else None)
        have = layer.cache.read(range(18))
        q, k, back, want = one_by_one(projections, layer, opened, x, flat, slots, table, lengths, counts)
        np.testing.assert_array_equal(y, want)
        codes, scales = oracle.encode(bf16_values(k)[:, 0])
        flat_codes = oracle.unpack(have["k_codes"]).reshape(-1, WIDTH)
        np.testing.assert_array_equal(flat_codes[slots], codes)
        np.testing.assert_array_equal(have["k_scales"].reshape(-1, WIDTH // 32)[slots], scales)
        latents = oracle.decode(codes, scales)
        first = np.concatenate([[0], np.cumsum(counts)])
        cached = [np.concatenate([c, latents[first[b]:first[b + 1]]]) for b, c in enumerate(cached)]
        keys = [c[:, None] for c in cached]
        out, lse, size = oracle.attend(bf16_values(q), keys, keys, lengths, np.array(counts), layer.scale, window, opened["sinks"])
        largest = np.maximum.reduce([np.abs(c).max(0) for c in cached])
        d = (56 * 2.0 ** -24 * (np.abs(bf16_values(q)).astype(np.float64) @ largest) * layer.scale + 2.0 ** -22)[..., None]
        limit = 2.0 ** -8 * (1 + 2.0 ** -8) * size + 2 * d * size + 2.0 ** -8 * np.abs(out)
        turned = oracle.heads(out, TABLE, flat, first=WIDTH - DIMS, dims=DIMS, inverse=True)
        pair = limit[..., WIDTH - DIMS:].reshape(*limit.shape[:-1], -1, 2).sum(-1).repeat(2, -1)   # |a c| + |b s| and no more
        error = np.concatenate([limit[..., :WIDTH - DIMS], pair + 2.0 ** -8 * (np.abs(turned[..., WIDTH - DIMS:]) + pair)], -1)
        assert np.all(np.abs(bf16_values(back) - turned) <= error + 1e-30)
    layer.close()


def test_captured_steps_follow_the_sequences(projections):
    """One captured step of a padded batch, replayed as its sequences grow, equals eager steps of a second layer."""
    rng = np.random.default_rng(9)
    opened = options(rng, max_tokens=4)
    ctx = projections.ctx
    table = rng.permutation(4 * 3).astype(np.int32).reshape(4, 3)
    captured, eager = (projections.open_cache(12, PAGE, TABLE, **opened) for _ in range(2))
    lengths, positions, slots = np.array([1, 1, 1, 0], np.int32), np.array([0, 0, 0, -1], np.int32), np.full(4, -1, np.int64)
    x = np.zeros((4, 5120), np.uint16)
    dev = [ctx.upload(a) for a in (x, positions, slots, table, lengths, x)]
    ptr = [d.ptr for d in dev]
    stream = ctx.stream()
    captured.step_device(ptr[0], 4, ptr[1], ptr[2], ptr[3], 3, ptr[4], 4, ptr[5], stream=stream)   # (the projections' scratch)
    ctx.sync()
    graph = Graph(ctx, stream, lambda: captured.step_device(ptr[0], 4, ptr[1], ptr[2], ptr[3], 3, ptr[4], 4, ptr[5], stream=stream))
    for at in range(20):
        x = bf16_bits(rng.standard_normal((4, 5120)).astype(np.float32))
        place = np.array([at, at, at, -1])
        slot = np.where(place < 0, -1, table[:, at // PAGE].astype(np.int64) * PAGE + at % PAGE)
        for d, a in zip(dev, (x, place.astype(np.int32), slot, table, np.maximum(place + 1, 0).astype(np.int32))):
            d.upload(a)
        ctx.sync()
        graph.launch()
        got = dev[5].download()
        want = eager.step(x[:3], place[:3], slot[:3], table[:3], place[:3] + 1)
        np.testing.assert_array_equal(got[:3], want)
    graph.close()
    ctx.destroy_stream(stream)
    for d in dev:
        d.free()
    captured.close(), eager.close()


def test_refusals_and_close(projections):
    rng = np.random.default_rng(1)
    layer = projections.open_cache(4, PAGE, TABLE, **options(rng, max_tokens=3, max_batch=2))
    x, at, table, lengths = np.zeros((2, 5120), np.uint16), np.zeros(2, int), np.array([[0], [1]]), np.ones(2, int)
    slots = np.array([0, PAGE])
    for args in ((x[:, :512], at, slots, table, lengths), (x.astype(np.float32), at, slots, table, lengths), (x[:1], at, slots, table, lengths),
                 (x, at + 600, slots, table, lengths), (x, at, slots * 0, table, lengths), (x, at, slots + 64, table, lengths),
                 (x, at, slots, table + 4, lengths), (x, at, slots, table, lengths + PAGE), (x, at, slots, table, lengths, [2, 1]),
                 (np.zeros((4, 5120), np.uint16), np.zeros(4, int), np.arange(4), table, lengths)):
        with pytest.raises(ValueError):
            layer.step(*args)
    assert layer.step(x, at, slots, table, lengths).shape == (2, 5120)
    layer.step_device(0, 0, 0, 0, 0, 1, 0, 0, 0)   # no tokens: nothing is launched
    with pytest.raises(ValueError):
        layer.step_device(1 << 20, 4, 1 << 20, 1 << 20, 1 << 20, 1, 1 << 20, 2, 1 << 20)
    layer.close()
    layer.close()
    with pytest.raises(RuntimeError):
        layer.step(x, at, slots, table, lengths)


def test_caches_close_with_the_runtime():
    rng = np.random.default_rng(2)
    arrays = {}
    for name, (rows, width) in dict(FP8_LAYOUT, wo_a=WO_A).items():
        w, s = fp8_weights(rng, rows, width, 32)
        arrays[f"layers.0.attn.{name}.weight"], arrays[f"layers.0.attn.{name}.scale"] = w, s
    proj = NativeProjections(arrays)
    with proj:
        layer = proj.open_cache(4, PAGE, TABLE, max_tokens=1, max_batch=1)
    assert proj.stats()["device_owned_bytes"] == 0
    with pytest.raises(RuntimeError):
        layer.step(np.zeros((1, 5120), np.uint16), [0], [0], [[0]], [1])
