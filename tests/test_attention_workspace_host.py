"""The workspace of attention, without a GPU: what its kernels can use for a cache's shape, and no more."""

import ctypes as C

import pytest

from vesper_amd import _lib

A = 1 << 20   # an aligned address that nothing reads


def need(width, value_width, heads, query_heads, tokens, batch):
    apart = A if width <= 256 else None
    cache = _lib.MxKv4(A, A, apart, apart, 4, 16, heads, width, value_width)
    return _lib.load().cdll.mx_kv4_workspace_bytes(C.c_void_p(0), C.byref(cache), query_heads, tokens, batch)


# (width, value width, workgroups, largest row tile): two parts of a workgroup's last units, FP32, with the rows' maxima and sums
@pytest.mark.parametrize("width,value_width,groups,rows", [(512, 512, 256, 64), (576, 512, 256, 64), (64, 64, 768, 128), (128, 128, 512, 128),
                                                          (256, 256, 256, 128)])
@pytest.mark.parametrize("tokens,batch", [(1, 1), (64, 64), (5000, 3)])
def test_parts_of_the_largest_tile_and_the_plan(width, value_width, groups, rows, tokens, batch):
    got = need(width, value_width, 1, 64, tokens, batch)
    parts = 2 * groups * rows * (4 * value_width + 8)
    plan = 4 * (batch + 1) + 8 * (tokens * 64 // 32 + batch + 1)     # at most, for the smallest tiles
    assert parts < got <= parts + plan + 20 * groups + 4 * 256
    assert got >= need(width, value_width, 1, 64, max(tokens // 2, 1), max(batch // 2, 1))   # a smaller call fits


def test_a_layer_of_latents_takes_67_mb():
    assert 67e6 < need(512, 512, 1, 64, 1, 1) < 68e6
