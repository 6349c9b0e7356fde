"""An attention layer over a cache without a GPU: what is refused before any device work."""

import types

import numpy as np
import pytest

from vesper_amd.attention import CachedAttention, rotation_table
from vesper_amd.projections import FP8_LAYOUT, NativeProjections

TABLE = rotation_table(16, 64)


def projections(**changes):
    """What CachedAttention looks at before it asks the device for anything."""
    return types.SimpleNamespace(**dict(dict(ctx=None, block=32, has_wo_a=True, layout=dict(FP8_LAYOUT)), **changes))


@pytest.mark.parametrize("change", [
    {"block": 128}, {"has_wo_a": False}, {"layout": {}}, {"layout": dict(FP8_LAYOUT, wq_b=(16384, 1280))},
    {"layout": dict(FP8_LAYOUT, wkv=(576, 5120))}, {"layout": dict(FP8_LAYOUT, wq_a=(1536, 5120))},
    {"layout": dict(FP8_LAYOUT, wkv=(512, 4096))}, {"layout": dict(FP8_LAYOUT, wo_b=(5120, 4096))}])
def test_other_projections_refused(change):
    with pytest.raises(ValueError, match="block-32|64 heads"):
        CachedAttention(projections(**change), 4, 64, TABLE, max_tokens=4, max_batch=2)


@pytest.mark.parametrize("change", [
    {"max_tokens": 0}, {"max_tokens": 1 << 20}, {"max_batch": 0}, {"scale": 0.0}, {"scale": float("nan")}, {"window": -1},
    {"q_norm": np.ones(512)}, {"kv_norm": np.ones(1280)}, {"sinks": np.ones(8)}, {"pages": 0}, {"page": 48}, {"table": None}])
def test_options_refused(change):
    args = dict(dict(pages=4, page=64, table=TABLE, max_tokens=4, max_batch=2), **change)
    with pytest.raises(ValueError):
        CachedAttention(projections(), args.pop("pages"), args.pop("page"), args.pop("table"), **args)


def test_a_runtime_that_is_not_open_has_no_cache():
    rng = np.random.default_rng(0)
    arrays = {"layers.0.attn.p.weight": rng.integers(0, 120, (64, 128), np.uint8),
              "layers.0.attn.p.scale": np.full((2, 4), 120, np.uint8)}
    with pytest.raises(RuntimeError, match="not open"):
        NativeProjections(arrays, layout={"p": (64, 128)}).open_cache(4, 64, TABLE, max_tokens=4, max_batch=2)
