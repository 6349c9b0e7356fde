"""Heads, 4-bit caches and their attention without a GPU: the oracle's pieces, and what the calls refuse before any
device work."""

import ctypes as C

import numpy as np
import pytest

from oracle import attention as oracle
from oracle.formats import bf16_bits, bf16_values
from vesper_amd import _lib
from vesper_amd.attention import HeadRotation, KVCache4, rotation_table

A = 1 << 20   # an aligned address that nothing reads: every call here is refused


def test_encode_keeps_blocks_in_range_and_rounds_to_the_nearest_code():
    rng = np.random.default_rng(1)
    x = bf16_values(bf16_bits((rng.standard_normal((64, 64)) * np.exp2(rng.integers(-20, 100, (64, 1)))).astype(np.float32)))
    x[0], x[1, :32] = 0, np.resize([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 6, -0.25], 32)
    codes, scales = oracle.encode(x)
    step = np.exp2(scales.astype(np.float64) - 127).repeat(32, -1)
    amax = np.abs(x.reshape(64, 2, 32)).max(-1).repeat(32, -1)
    assert np.all(amax <= 6 * step)
    assert np.all((amax > 3 * step) | (amax < 1e-4))      # half the scale would not do
    y = np.abs(x) / step
    want = (y > .25).astype(int) + (y >= .75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)
    np.testing.assert_array_equal(codes & 7, want)
    np.testing.assert_array_equal(codes >> 3, np.signbit(x))
    np.testing.assert_array_equal(oracle.unpack(oracle.pack(codes)), codes)


def test_encode_marks_blocks_that_are_not_finite_and_caps_the_scale():
    x = np.ones((3, 96))
    x[0, 5], x[1, 40] = np.inf, np.nan
    x[2, :32] = bf16_values(np.array([0x7F7F], np.uint16))[0]
    codes, scales = oracle.encode(x)
    assert scales.tolist()[0][0] == 255 and scales.tolist()[1][1] == 255 and scales[2, 0] == 252
    assert np.all(scales[:, 2] == scales[0, 1]) and np.isnan(oracle.decode(codes, scales)[0, :32]).all()
    np.testing.assert_array_equal(oracle.decode(codes, scales)[2, :32], 6 * 2.0 ** 125)


def test_gradients_are_the_differences_of_the_formula():
    rng = np.random.default_rng(2)
    table, pos = rotation_table(9, 16), np.array([3, 8, 0])
    for style in ("pairs", "halves"):
        args = dict(norm=24, first=16, dims=16, style=style, eps=1e-3)
        x, dy, w = rng.standard_normal((3, 2, 40)), rng.standard_normal((3, 2, 40)), rng.uniform(.5, 1.5, 24)
        dx, dw = oracle.heads_backward(dy, x, table, pos, weight=w, **args)
        for _ in range(20):
            d, e = rng.standard_normal(x.shape), rng.standard_normal(24)
            f = lambda s: np.sum(dy * oracle.heads(x + s * d, table, pos, weight=w + s * e, **args))  # noqa: E731
            slope = (f(1e-5) - f(-1e-5)) / 2e-5
            assert abs(slope - np.sum(dx * d) - np.sum(dw * e)) <= 1e-7 * (1 + abs(slope))


def test_rotation_table_in_far_positions():
    t = rotation_table(1 << 20, 8, base=1e6)
    angle = (2 ** 20 - 1) * np.array([1.0, 1e6 ** -0.25, 1e6 ** -0.5, 1e6 ** -0.75])
    np.testing.assert_allclose(t[-1], np.concatenate([np.cos(angle), np.sin(angle)]), atol=2 ** -24)
    for bad in ((0, 8), (8, 7), (8, 0)):
        with pytest.raises(ValueError):
            rotation_table(*bad)


def test_oracle_attention_of_windows_sinks_and_empty_rows():
    k = [np.zeros((4, 1, 2)), np.zeros((0, 1, 2))]
    v = [np.arange(8.0).reshape(4, 1, 2), np.zeros((0, 1, 2))]
    out, lse, _ = oracle.attend(np.zeros((3, 1, 2)), k, v, [4, 0], [2, 1], 1.0, window=2)
    np.testing.assert_allclose(out[:, 0], [[3, 4], [5, 6], [0, 0]])
    np.testing.assert_allclose(lse[:2, 0], np.log(2))
    assert lse[2, 0] == -np.inf
    out, _, _ = oracle.attend(np.zeros((1, 1, 2)), k[:1], v[:1], [4], [1], 1.0, sinks=np.log([4.0]))
    np.testing.assert_allclose(out[0, 0], [1.5, 2])


# -- refusals of the C entry points ------------------------------------------------------------------------

CTX = C.c_void_p(0)   # a null context is the last refusal: MX_ERR_STATE


def rotation(**change):
    fields = dict(table=A, table_positions=16, positions=A, width=128, norm=128, first=64, dims=64, style=0, inverse=0, eps=1e-6)
    return _lib.MxRotation(**{**fields, **change})


def status(fn, *args):
    return getattr(_lib.load().cdll, fn)(*args)


@pytest.mark.parametrize("change", [
    dict(width=0), dict(width=12), dict(width=4104), dict(norm=-8), dict(norm=12), dict(norm=136), dict(dims=-8), dict(dims=12),
    dict(first=4), dict(first=-8), dict(first=72), dict(first=2 ** 31 - 8), dict(style=2), dict(style=1, dims=24), dict(inverse=2), dict(eps=-1.0),
    dict(eps=float("nan")), dict(eps=float("inf")), dict(table=None), dict(table=A + 4), dict(positions=None),
    dict(positions=A + 2), dict(table_positions=0)])
def test_rotations_refused(change):
    heads = _lib.MxHeads(A, 1024, 8, None, A, 1024)
    grads = _lib.MxHeadsGrad(A, 1024, 8, None, A, 1024, A, 1024, None)
    rows = _lib.MxKv4Append(A, 128, A, 128, 0, 1, A, None, None, None)
    for args in (("mx_rotate_heads", CTX, C.byref(heads), 1, 1, C.byref(rotation(**change)), 0, 0, None),
                 ("mx_rotate_heads_backward", CTX, C.byref(grads), 1, 1, C.byref(rotation(**change)), 0, None, 0, None),
                 ("mx_kv4_append", CTX, C.byref(cache()), C.byref(rows), C.byref(rotation(**change)), None)):
        assert status(*args) == _lib.MX_ERR_INVALID


@pytest.mark.parametrize("heads,n,tokens,types", [
    (_lib.MxHeads(None, 1024, 8, None, A, 1024), 1, 1, (0, 0)), (_lib.MxHeads(A, 1024, 8, None, None, 1024), 1, 1, (0, 0)),
    (_lib.MxHeads(A, 1023, 8, None, A, 1024), 1, 1, (0, 0)), (_lib.MxHeads(A, 1024, 8, None, A, 1016), 1, 1, (0, 0)),
    (_lib.MxHeads(A, 1024, 0, None, A, 1024), 1, 1, (0, 0)), (_lib.MxHeads(A, 1024, -1, None, A, 1024), 1, 1, (0, 0)),
    (_lib.MxHeads(A + 1, 1024, 8, None, A, 1024), 1, 1, (0, 0)), (_lib.MxHeads(A, 1024, 8, A + 2, A, 1024), 1, 1, (0, 0)),
    (_lib.MxHeads(A, 1024, 8, None, A, 2048), 1, 1, (0, 0)), (_lib.MxHeads(A, 1024, 8, None, A, 1024), 1, 1, (1, 0)),
    (_lib.MxHeads(A, 1024, 8, None, A, 1024), 1, 1, (2, 2)), (_lib.MxHeads(A, 1024, 8, None, A, 1024), 0, 1, (0, 0)),
    (_lib.MxHeads(A, 1024, 8, None, A, 1024), 3, 1, (0, 0)), (_lib.MxHeads(A, 1024, 8, None, A, 1024), 1, -1, (0, 0)),
    (_lib.MxHeads(A, 1024, 8, None, A, 1024), 1, 2 ** 20 + 1, (0, 0)),
    (_lib.MxHeads(A, 1 << 21, 1 << 12, None, A, 1 << 21), 1, 1 << 20, (0, 0))])
def test_heads_refused(heads, n, tokens, types):
    array = (_lib.MxHeads * 3)(heads, heads, heads)
    assert status("mx_rotate_heads", CTX, array, n, tokens, C.byref(rotation()), *types, None) == _lib.MX_ERR_INVALID


def test_heads_gradients_refused():
    def grad(**change):
        fields = dict(x=A, x_stride=1024, heads=8, weight=None, dy=A, dy_stride=1024, dx=A, dx_stride=1024, dweight=None)
        return _lib.MxHeadsGrad(**{**fields, **change})
    need = _lib.load().cdll.mx_rotate_heads_workspace_bytes(128)
    assert need > 0 and _lib.load().cdll.mx_rotate_heads_workspace_bytes(-1) == 0
    call = lambda g, work=(A, need), rot=rotation(): status(  # noqa: E731
        "mx_rotate_heads_backward", CTX, C.byref(g), 1, 1, C.byref(rot), 0, *work, None)
    assert call(grad(dweight=A)) == _lib.MX_ERR_STATE      # all else is in order
    assert call(grad(x=None, x_stride=0), rot=rotation(norm=0)) == _lib.MX_ERR_STATE
    for g in (grad(x=None), grad(dy=None), grad(dx=None), grad(dx_stride=2048), grad(x_stride=2048), grad(dy_stride=1016)):
        assert call(g) == _lib.MX_ERR_INVALID
    for work in ((None, need), (A, need - 1), (A + 8, need)):
        assert call(grad(dweight=A), work) == _lib.MX_ERR_INVALID
    assert call(grad(dweight=A), rot=rotation(norm=0)) == _lib.MX_ERR_INVALID


def cache(**change):
    fields = dict(k_codes=A, k_scales=A, v_codes=A, v_scales=A, pages=4, page=16, heads=1, width=128, value_width=128)
    return _lib.MxKv4(**{**fields, **change})


BAD_CACHES = [dict(page=8), dict(page=24), dict(page=2048), dict(pages=0), dict(heads=0), dict(heads=1025), dict(width=96, value_width=96),
              dict(width=512, value_width=512), dict(value_width=64), dict(v_codes=None), dict(v_scales=None), dict(k_codes=None),
              dict(k_scales=None), dict(k_codes=A + 8), dict(v_scales=A + 4),
              dict(v_codes=None, v_scales=None), dict(v_codes=None, v_scales=None, width=576, value_width=576)]


@pytest.mark.parametrize("change", BAD_CACHES)
def test_caches_refused(change):
    rows = _lib.MxKv4Append(A, 1024, A, 1024, 0, 1, A, None, None, None)
    query = _lib.MxKv4Attend(A, 1024, 1, 1, 1, None, A, 1, A, 1.0, 0, None, A, 1024, None)
    c = cache(**change)
    assert status("mx_kv4_append", CTX, C.byref(c), C.byref(rows), None, None) == _lib.MX_ERR_INVALID
    assert status("mx_kv4_attend", CTX, C.byref(c), C.byref(query), A, 1 << 40, None) == _lib.MX_ERR_INVALID
    assert status("mx_kv4_workspace_bytes", CTX, C.byref(c), 1, 1, 1) == 0


@pytest.mark.parametrize("change", [
    dict(k=None), dict(slots=None), dict(v=None), dict(type=2), dict(tokens=-1), dict(tokens=2 ** 20 + 1), dict(k_stride=127),
    dict(v_stride=64), dict(k=A + 1), dict(slots=A + 4), dict(weight=A + 2), dict(k_rounded=A + 8), dict(v_rounded=A + 2)])
def test_appends_refused(change):
    fields = dict(k=A, k_stride=128, v=A, v_stride=128, type=0, tokens=1, slots=A, weight=None, k_rounded=None, v_rounded=None)
    call = lambda r: status("mx_kv4_append", CTX, C.byref(cache()), C.byref(r), None, None)  # noqa: E731
    assert call(_lib.MxKv4Append(**fields)) == _lib.MX_ERR_STATE
    assert call(_lib.MxKv4Append(**{**fields, **change})) == _lib.MX_ERR_INVALID


def test_an_append_of_latents_takes_no_values_and_a_rotation_of_its_width():
    c = cache(v_codes=None, v_scales=None, width=512, value_width=512)
    for v, rounded in ((A, None), (None, A)):
        rows = _lib.MxKv4Append(A, 512, v, 512, 0, 1, A, None, None, rounded)
        assert status("mx_kv4_append", CTX, C.byref(c), C.byref(rows), None, None) == _lib.MX_ERR_INVALID
    rows = _lib.MxKv4Append(A, 512, None, 0, 0, 1, A, None, None, None)
    assert status("mx_kv4_append", CTX, C.byref(c), C.byref(rows), C.byref(rotation()), None) == _lib.MX_ERR_INVALID


@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(table=None), dict(lengths=None), dict(heads=0), dict(heads=3), dict(tokens=-1),
    dict(tokens=2 ** 20 + 1), dict(tokens=5), dict(batch=-1), dict(batch=0), dict(batch=2 ** 16 + 1), dict(columns=0), dict(columns=2 ** 27),
    dict(q_stride=504), dict(q_stride=516), dict(out_stride=504), dict(out_stride=514), dict(q=A + 8), dict(out=A + 2),
    dict(window=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-1.0), dict(lse=A + 2),
    dict(sinks=A + 1), dict(q_first=A + 2), dict(lengths=A + 2), dict(table=A + 2)])
def test_attends_refused(change):
    fields = dict(q=A, q_stride=512, heads=4, tokens=4, batch=2, q_first=None, table=A, columns=2, lengths=A, scale=1.0, window=0,
                  sinks=None, out=A, out_stride=512, lse=None)
    c = cache(heads=2)
    need = status("mx_kv4_workspace_bytes", CTX, C.byref(c), 4, 4, 2)
    assert need > 0
    call = lambda q, work=(A, need): status("mx_kv4_attend", CTX, C.byref(c), C.byref(q), *work, None)  # noqa: E731
    good = _lib.MxKv4Attend(**fields)
    assert call(good) == _lib.MX_ERR_STATE
    assert call(_lib.MxKv4Attend(**{**fields, **change})) == _lib.MX_ERR_INVALID
    for work in ((None, need), (A, need - 1), (A + 8, need)):
        assert call(good, work) == _lib.MX_ERR_INVALID


# -- refusals of the Python classes --------------------------------------------------------------------------

class NoDevice:
    """A context whose every use is a mistake of the caller's checks."""
    lib = property(lambda self: pytest.fail("a refused call reached the library"))

    def upload(self, *_):
        pytest.fail("a refused call reached the device")
    empty = malloc = _h = upload


@pytest.mark.parametrize("kwargs", [
    dict(width=12), dict(width=0), dict(width=8192), dict(width=64, norm=72), dict(width=64, norm=4), dict(width=64, dims=4),
    dict(width=64, dims=8, style="halves"), dict(width=64, dims=8, style="thirds"), dict(width=64, dims=32, first=40),
    dict(width=64, dims=32, first=4), dict(width=64, norm=64, eps=-1.0), dict(width=64, norm=64, eps=float("nan")),
    dict(width=64, dims=32), dict(width=64, dims=32, table=np.zeros((4, 16))), dict(width=64, dims=32, table=np.full((4, 32), np.inf)),
    dict(width=64, dims=32, table=np.zeros((0, 32)))])
def test_head_rotations_refused(kwargs):
    with pytest.raises(ValueError):
        HeadRotation(NoDevice(), **kwargs)


@pytest.mark.parametrize("args,kwargs", [
    ((4, 16, 1, 96), {}), ((4, 16, 1, 512), {}), ((4, 16, 1, 128, 128), {}), ((4, 16, 1, 576, 576), {}), ((4, 8, 1, 64), {}),
    ((4, 48, 1, 64), {}), ((0, 16, 1, 64), {}), ((4, 16, 0, 64), {}), ((4, 16, 2, 64), dict(query_heads=3)),
    ((4, 16, 1, 64), dict(max_tokens=0)), ((4, 16, 1, 64), dict(max_batch=0)), ((4, 16, 1, 64), dict(max_batch=2 ** 16 + 1))])
def test_kv_caches_refused(args, kwargs):
    with pytest.raises(ValueError):
        KVCache4(NoDevice(), *args, **{**dict(query_heads=4, max_tokens=8, max_batch=8), **kwargs})
