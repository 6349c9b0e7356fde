"""What stands between the attention projections and the output projection: heads normalized and rotated, a paged
key/value cache in 4 bits, and the attention that reads it (the reference's norm_*, rope_* and window kernels run one
query at a time, src/vesper/kernels/normalization_probe.cu:4-86; its cache keeps BF16 rows).

HeadRotation   y = rotation(weight * x / rms(x)) of every head, and its gradients
KVCache4       pages of E2M1 codes with an E8M0 scale per 32 values: append (normalized and rotated on the way), attend
CachedAttention  the block-32 projections' attention over a cache (NativeProjections.open_cache): wq_a and wq_b with their
               norms, the rotation, wkv into the cache, attention, the rotation back, wo_a, wo_b

The *_device methods take device pointers and do not synchronise; the others take and return host arrays (BF16 as uint16
bits, or FP32). A HeadRotation and a KVCache4 have one workspace, a CachedAttention one set of buffers: calls of one object
must not overlap on different streams. Calls from several threads take turns, each with all its launches, and close waits for
them.
"""

from __future__ import annotations

import ctypes as C
import math
import threading

import numpy as np

from . import _lib
from .dispatch import host_rows, row_type
from .projections import GROUPED_MAX_TOKENS, WO_A, WO_A_GROUPS, validate_values

MAX_TOKENS, MAX_WIDTH, MAX_BATCH, MAX_HEADS = 1 << 20, 4096, 1 << 16, 1 << 16
APART_WIDTHS, LATENT_WIDTHS = (64, 128, 256), ((512, 512), (576, 512))


def _count(value, most: int, what: str) -> int:
    """A number that a call hands to the library in 32 bits."""
    if not 0 <= value <= most:
        raise ValueError(f"{what} must be in [0, {most}]")
    return int(value)


def rotation_table(positions: int, dims: int, base: float = 10000.0, scaling: float = 1.0) -> np.ndarray:
    """FP32 [positions, dims]: dims / 2 cosines of the angles scaling * p * base^(-2 i / dims), then their sines,
    computed in 64 bits."""
    if positions < 1 or dims < 2 or dims % 2 or not base > 0:
        raise ValueError("a table needs positions, an even number of dims and a positive base")
    angle = np.arange(positions, dtype=np.float64)[:, None] * scaling * base ** (-np.arange(0, dims, 2) / dims)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def _window(window) -> int:
    """Of 2^31 positions and more, which are all that a length can have, as 2^31 - 1."""
    if window < 0:
        raise ValueError("window must not be negative")
    return min(int(window), 2 ** 31 - 1)


class HeadRotation:
    """The norm and rotation of heads of `width` values: the first `norm` values are normalized, the `dims` values from
    `first` on (None: the last) turned by `table` (rotation_table; FP32 [positions, dims])."""

    def __init__(self, ctx: _lib.Context, width: int, norm: int = 0, dims: int = 0, first: int | None = None,
                 style: str = "pairs", eps: float = 1e-6, table=None):
        if style not in _lib.MX_ROTATE:
            raise ValueError("rotation style must be pairs or halves")
        first = width - dims if first is None else first
        unit = 16 if style == "halves" else 8
        if not 8 <= width <= MAX_WIDTH or width % 8 or not 0 <= norm <= width or norm % 8:
            raise ValueError(f"width must be a multiple of 8 in [8, {MAX_WIDTH}] and norm one up to it")
        if dims < 0 or dims % unit or first < 0 or first % 8 or first + dims > width:
            raise ValueError(f"rotated values must be a multiple of {unit} within the head, from a multiple of 8 on")
        if not (math.isfinite(eps) and eps >= 0):
            raise ValueError("eps must be finite and not negative")
        if dims:
            table = np.ascontiguousarray(table, np.float32)
            if table.ndim != 2 or table.shape[0] < 1 or table.shape[1] != dims or not np.isfinite(table).all():
                raise ValueError(f"the rotation's table must be finite FP32 [positions, {dims}]")
        self.lock = threading.RLock()
        self.ctx, self.width, self.norm, self.first, self.dims = ctx, int(width), int(norm), int(first), int(dims)
        self.style, self.eps = _lib.MX_ROTATE[style], float(eps)
        self.positions = table.shape[0] if dims else 0
        self.table = ctx.upload(table) if dims else None
        self.workspace_bytes = int(ctx.lib.cdll.mx_rotate_heads_workspace_bytes(self.norm))
        self.workspace = None

    def close(self):
        with self.lock:
            for name in ("table", "workspace"):
                held = getattr(self, name)
                if held is not None:
                    setattr(self, name, None)
                    held.free()
            self.ctx = None

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def _open(self):
        if self.ctx is None:
            raise RuntimeError("the rotation is closed")
        return self.ctx._h()

    def struct(self, positions_ptr=None, inverse: bool = False) -> _lib.MxRotation:
        self._open()
        return _lib.MxRotation(_lib.ptr(self.table), self.positions, _lib.ptr(positions_ptr), self.width, self.norm,
                               self.first, self.dims, self.style, int(bool(inverse)), self.eps)

    def set(self, x_ptr, heads, y_ptr, weight_ptr=None, x_stride=None, y_stride=None) -> _lib.MxHeads:
        """`heads` heads of every token at x_ptr, to y_ptr (strides in values between tokens; None: contiguous)."""
        heads, ptr = _count(heads, MAX_HEADS, "heads"), _lib.ptr
        own = heads * self.width
        return _lib.MxHeads(ptr(x_ptr), own if x_stride is None else x_stride, heads, ptr(weight_ptr), ptr(y_ptr),
                            own if y_stride is None else y_stride)

    def grad(self, x_ptr, heads, dy_ptr, dx_ptr, weight_ptr=None, dweight_ptr=None, x_stride=None, dy_stride=None,
             dx_stride=None) -> _lib.MxHeadsGrad:
        heads, ptr = _count(heads, MAX_HEADS, "heads"), _lib.ptr
        own = heads * self.width
        return _lib.MxHeadsGrad(ptr(x_ptr), own if x_stride is None else x_stride, heads, ptr(weight_ptr), ptr(dy_ptr),
                                own if dy_stride is None else dy_stride, ptr(dx_ptr), own if dx_stride is None else dx_stride,
                                ptr(dweight_ptr))

    # -- device pointers in and out, no host synchronisation ---------------------------------------
    def apply_device(self, sets, tokens: int, positions_ptr=None, x_dtype: str = "bf16", y_dtype: str | None = None,
                     inverse: bool = False, stream=None):
        """One or two `set`s (queries, and keys with weights of their own) in one launch."""
        with self.lock:
            rotation = self.struct(positions_ptr, inverse)
            array = (_lib.MxHeads * len(sets))(*sets)
            self.ctx.lib.rotate_heads(self.ctx._h(), array, len(sets), _count(tokens, MAX_TOKENS, "tokens"), C.byref(rotation),
                                      row_type(x_dtype), row_type(y_dtype or x_dtype), _lib._stream(stream))

    def open_gradients(self):
        """The workspace of the weights' gradients; allocated by the first call that needs it unless opened before (a
        call inside a stream capture cannot allocate)."""
        with self.lock:
            self._open()
            if self.workspace is None and self.workspace_bytes:
                self.workspace = self.ctx.empty((self.workspace_bytes,), np.uint8)

    def backward_device(self, grads, tokens: int, positions_ptr=None, dtype: str = "bf16", inverse: bool = False,
                        stream=None):
        """The gradients of apply_device(inverse) for one or two `grad`s, each with a dweight of its own (the sum of both is
        the gradient of a weight that they share). Calls that ask for dweight share a workspace: they must not overlap on
        different streams."""
        with self.lock:
            rotation = self.struct(positions_ptr, inverse)
            if any(g.dweight for g in grads):
                self.open_gradients()
            array = (_lib.MxHeadsGrad * len(grads))(*grads)
            self.ctx.lib.rotate_heads_backward(self.ctx._h(), array, len(grads), _count(tokens, MAX_TOKENS, "tokens"),
                                               C.byref(rotation), row_type(dtype), _lib.ptr(self.workspace),
                                               self.workspace_bytes, _lib._stream(stream))

    # -- host arrays -------------------------------------------------------------------------------
    def _host(self, x, what):
        x = np.asarray(x)
        if x.ndim != 3 or x.shape[2] != self.width or not 0 <= x.shape[0] <= MAX_TOKENS or x.shape[1] < 1:
            raise ValueError(f"{what} must be [T, heads, {self.width}]")
        flat, dtype = host_rows(x.reshape(x.shape[0], x.shape[1] * self.width) if x.size else
                                np.zeros((0, x.shape[1] * self.width), x.dtype))
        return flat, dtype, x.shape[:2]

    def _positions(self, positions, tokens):
        if not self.dims:
            return None
        positions = np.asarray(positions)
        if positions.dtype not in (np.dtype(np.int32), np.dtype(np.int64)) or positions.shape != (tokens,):
            raise ValueError(f"positions must be an integer array [{tokens}]")
        if positions.size and (positions.min() < -1 or positions.max() >= self.positions):
            raise ValueError(f"positions must be in [0, {self.positions}), or -1 for no token")
        return positions.astype(np.int32)

    def _weight(self, weight):
        if weight is None:
            return None
        weight = np.ascontiguousarray(weight, np.float32)
        if weight.shape != (self.norm,) or not self.norm:
            raise ValueError(f"the norm's weight must be [{self.norm}]")
        return weight

    def apply(self, x, positions=None, weight=None, inverse: bool = False) -> np.ndarray:
        """[T, heads, width] of x, in its type; rows of no token (position -1) as they were."""
        self._open()
        flat, dtype, (t, heads) = self._host(x, "x")
        dev = []
        try:
            for a in (flat, self._positions(positions, t), self._weight(weight)):
                dev.append(None if a is None else self.ctx.upload(a))
            s = self.set(dev[0], heads, dev[0], dev[2])
            self.apply_device([s], t, dev[1], dtype, inverse=inverse)
            return dev[0].download().reshape(t, heads, self.width)
        finally:
            for d in dev:
                if d is not None:
                    d.free()

    def backward(self, dy, x, positions=None, weight=None, inverse: bool = False) -> dict:
        """{"dx" [T, heads, width], and with norm "dweight" [norm]}."""
        self._open()
        dy, dtype, (t, heads) = self._host(dy, "dy")
        x, x_dtype, shape = self._host(x, "x")
        if x_dtype != dtype or shape != (t, heads):
            raise ValueError("x and its output's gradient must have one type and shape")
        dev = []
        try:
            for a in (dy, x, self._positions(positions, t), self._weight(weight),
                      np.zeros(self.norm, np.float32) if self.norm else None):
                dev.append(None if a is None else self.ctx.upload(a))
            grad = self.grad(dev[1], heads, dev[0], dev[1], dev[3], dev[4])
            self.backward_device([grad], t, dev[2], dtype, inverse)
            out = {"dx": dev[1].download().reshape(t, heads, self.width)}
            if self.norm:
                out["dweight"] = dev[4].download()
            return out
        finally:
            for d in dev:
                if d is not None:
                    d.free()


class KVCache4:
    """`pages` pages of `page` tokens for `heads` key heads. value_width None: values apart from the keys, as wide as
    they are; else latents, whose values are the first value_width values of the key. query_heads, max_tokens (query rows
    of one attend call) and max_batch size the workspace."""

    def __init__(self, ctx: _lib.Context, pages: int, page: int, heads: int, width: int, value_width: int | None = None,
                 *, query_heads: int, max_tokens: int, max_batch: int):
        if value_width is None and width not in APART_WIDTHS:
            raise ValueError(f"keys with values apart must be {APART_WIDTHS} wide")
        if value_width is not None and (width, value_width) not in LATENT_WIDTHS:
            raise ValueError(f"latents and their values must be {LATENT_WIDTHS} wide")
        if not 16 <= page <= 1024 or page & (page - 1):
            raise ValueError("a page must be a power of two of tokens in [16, 1024]")
        if pages < 1 or not 1 <= heads <= 1024 or not 1 <= query_heads <= MAX_HEADS or query_heads % heads:
            raise ValueError(f"a cache needs pages, and query heads that are a multiple of its key heads, {MAX_HEADS} at most")
        if not 1 <= max_tokens <= MAX_TOKENS or not 1 <= max_batch <= MAX_BATCH:
            raise ValueError(f"max_tokens in [1, {MAX_TOKENS}] and max_batch in [1, {MAX_BATCH}] required")
        self.ctx, self.pages, self.page, self.heads = ctx, int(pages), int(page), int(heads)
        self.width, self.apart = int(width), value_width is None
        self.value_width = self.width if self.apart else int(value_width)
        self.query_heads, self.max_tokens, self.max_batch = int(query_heads), int(max_tokens), int(max_batch)
        self.lock, self._owned = threading.Lock(), []
        try:
            for w in (self.width, self.value_width) if self.apart else (self.width,):
                for bytes_ in (w // 2, -(-w // 128) * 4):
                    self._owned.append(ctx.empty((self.pages, self.heads, self.page, bytes_), np.uint8))
            arrays = self._owned + [None] * (4 - len(self._owned))
            self.struct = _lib.MxKv4(*map(_lib.ptr, arrays), self.pages, self.page, self.heads, self.width,
                                     self.value_width)
            self.workspace_bytes = int(ctx.lib.cdll.mx_kv4_workspace_bytes(
                ctx._h(), C.byref(self.struct), self.query_heads, self.max_tokens, self.max_batch))
            if not self.workspace_bytes:
                raise ValueError(ctx.lib.last_error())
            self.workspace = ctx.empty((self.workspace_bytes,), np.uint8)
            self._owned.append(self.workspace)
        except BaseException:
            self.close()
            raise

    def close(self):
        with self.lock:
            while self._owned:
                self._owned.pop().free()

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def _open(self):
        if not self._owned:
            raise RuntimeError("the cache is closed")
        return self.ctx._h()

    # -- device pointers in and out, no host synchronisation ---------------------------------------
    def append_device(self, k_ptr, slots_ptr, tokens: int, v_ptr=None, rotation: HeadRotation | None = None,
                      positions_ptr=None, weight_ptr=None, dtype: str = "bf16", k_stride=None, v_stride=None,
                      k_rounded_ptr=None, v_rounded_ptr=None, stream=None):
        """Keys [T, heads, width] (through `rotation`) and values into device int64 slots [T] (page * self.page + place;
        outside the cache: not stored), and the BF16 values that the codes stand for where asked."""
        with self.lock:
            handle, ptr = self._open(), _lib.ptr
            turned = None if rotation is None else rotation.struct(positions_ptr)
            if rotation is not None and rotation.ctx is not self.ctx and rotation.ctx.ordinal != self.ctx.ordinal:
                raise ValueError(f"the rotation is on device {rotation.ctx.ordinal}, the cache on {self.ctx.ordinal}")
            rows = _lib.MxKv4Append(ptr(k_ptr), self.heads * self.width if k_stride is None else k_stride, ptr(v_ptr),
                                    self.heads * self.value_width if v_stride is None else v_stride, row_type(dtype),
                                    _count(tokens, MAX_TOKENS, "tokens"), ptr(slots_ptr), ptr(weight_ptr),
                                    ptr(k_rounded_ptr), ptr(v_rounded_ptr))
            self.ctx.lib.kv4_append(handle, C.byref(self.struct), C.byref(rows), None if turned is None else C.byref(turned),
                                    _lib._stream(stream))

    def attend_device(self, q_ptr, tokens: int, table_ptr, columns: int, lengths_ptr, batch: int, out_ptr, scale: float,
                      q_first_ptr=None, window: int = 0, sinks_ptr=None, lse_ptr=None, q_stride=None, out_stride=None,
                      stream=None):
        """out [T, query_heads, value_width] BF16 of q [T, query_heads, width] BF16: tokens / batch query rows of each
        sequence, or those that device int32 q_first [batch + 1] gives."""
        with self.lock:
            handle, ptr = self._open(), _lib.ptr
            if not 0 <= tokens <= self.max_tokens or not 0 <= batch <= self.max_batch:
                raise ValueError(f"the cache was opened for {self.max_tokens} query rows of {self.max_batch} sequences a call")
            query = _lib.MxKv4Attend(ptr(q_ptr), self.query_heads * self.width if q_stride is None else q_stride,
                                     self.query_heads, int(tokens), int(batch), ptr(q_first_ptr), ptr(table_ptr),
                                     _count(columns, (1 << 30) // self.page, "columns"),
                                     ptr(lengths_ptr), float(scale), _window(window), ptr(sinks_ptr), ptr(out_ptr),
                                     self.query_heads * self.value_width if out_stride is None else out_stride, ptr(lse_ptr))
            self.ctx.lib.kv4_attend(handle, C.byref(self.struct), C.byref(query), self.workspace.ptr, self.workspace_bytes,
                                    _lib._stream(stream))

    # -- host arrays -------------------------------------------------------------------------------
    def _rows(self, x, width, what, heads):
        x = np.asarray(x)
        if x.dtype not in (np.dtype(np.uint16), np.dtype(np.float32)) or x.ndim != 3 or x.shape[1:] != (heads, width) \
                or x.shape[0] > MAX_TOKENS:
            raise ValueError(f"{what} must be BF16 storage bits or FP32 values [T, {heads}, {width}]")
        return np.ascontiguousarray(x), "bf16" if x.dtype == np.uint16 else "f32"

    def _slots(self, slots, tokens):
        slots = np.asarray(slots)
        if slots.dtype not in (np.dtype(np.int32), np.dtype(np.int64)) or slots.shape != (tokens,):
            raise ValueError(f"slots must be an integer array [{tokens}]")
        stored = slots[slots >= 0]
        if stored.size and stored.max() >= self.pages * self.page:
            raise ValueError(f"slots must be in [0, {self.pages * self.page}), or negative for none")
        if np.unique(stored).size != stored.size:
            raise ValueError("two tokens name one slot")
        return np.ascontiguousarray(slots, np.int64)

    def _sequences(self, table, lengths, counts, t, window=0):
        """The int32 arrays of `t` query rows' sequences: pages, lengths and, with counts, first rows. Pages of which no row
        sees a token, behind the length or before the windows, may have any number."""
        table, lengths = np.asarray(table), np.asarray(lengths)
        b = lengths.shape[0] if lengths.ndim == 1 else -1
        if (b < 0 or table.ndim != 2 or table.shape[0] != b or table.shape[1] < 1
                or any(a.dtype not in (np.dtype(np.int32), np.dtype(np.int64)) for a in (table, lengths))):
            raise ValueError("table must be an integer array [B, columns] and lengths one [B]")
        if b and (lengths.min() < 0 or lengths.max() > table.shape[1] * self.page):
            raise ValueError("lengths must fit their pages")
        first, rows = None, np.full(b, t // max(b, 1))
        if counts is not None:
            counts = np.asarray(counts)
            if counts.shape != (b,) or counts.dtype.kind not in "iu" or (b and counts.min() < 0) or counts.sum() > t:
                raise ValueError(f"counts must be {b} numbers of query rows, {t} in all")
            rows, first = counts.astype(np.int64), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        elif t % max(b, 1) or (t and not b):
            raise ValueError("query rows do not divide among the sequences")
        page = np.arange(table.shape[1]) * self.page
        used = page < lengths[:, None]
        if window:   # from the first row's first token on
            used &= page + self.page > (lengths.astype(np.int64) - rows + 1 - _window(window))[:, None]
        if np.any(used & ((table < 0) | (table >= self.pages))):
            raise ValueError(f"page numbers in use must be in [0, {self.pages})")
        return np.ascontiguousarray(table, np.int32), np.ascontiguousarray(lengths, np.int32), first

    def append(self, k, slots, v=None, rotation: HeadRotation | None = None, positions=None, weight=None) -> dict:
        """Stores the tokens; {"k" [T, heads, width], and "v"}: BF16 bits of what the codes stand for (zero where a token
        is not stored)."""
        self._open()
        k, dtype = self._rows(k, self.width, "keys", self.heads)
        t = k.shape[0]
        if (v is not None) != self.apart:
            raise ValueError("values are given where the cache holds them apart from the keys")
        if v is not None:
            v, v_dtype = self._rows(v, self.value_width, "values", self.heads)
            if v_dtype != dtype or v.shape[0] != t:
                raise ValueError("keys and values must be of one type and as many tokens")
        slots = self._slots(slots, t)
        if rotation is None and (positions is not None or weight is not None):
            raise ValueError("positions and weight go with a rotation")
        if rotation is not None and rotation.width != self.width:
            raise ValueError(f"the rotation is of {rotation.width} values, the keys of {self.width}")
        inputs = [k, v, slots, None if rotation is None else rotation._positions(positions, t),
                  None if rotation is None else rotation._weight(weight)]
        outputs = [np.zeros(k.shape, np.uint16), None if v is None else np.zeros(v.shape, np.uint16)]
        dev = []
        try:
            for a in inputs + outputs:
                dev.append(None if a is None else self.ctx.upload(a))
            self.append_device(dev[0], dev[2], t, dev[1], rotation, dev[3], dev[4], dtype, k_rounded_ptr=dev[5],
                               v_rounded_ptr=dev[6])
            out = {"k": dev[5].download()}
            if v is not None:
                out["v"] = dev[6].download()
            return out
        finally:
            for d in dev:
                if d is not None:
                    d.free()

    def attend(self, q, table, lengths, scale: float, counts=None, window: int = 0, sinks=None) -> dict:
        """{"out" [T, query_heads, value_width] BF16 bits, "lse" [T, query_heads]}: q [T, query_heads, width] BF16 bits,
        table [B, columns] pages, lengths [B]; counts [B] query rows of each sequence (None: as many of each)."""
        self._open()
        q, dtype = self._rows(q, self.width, "q", self.query_heads)
        if dtype != "bf16":
            raise ValueError("q must be BF16 storage bits")
        t = q.shape[0]
        table, lengths, first = self._sequences(table, lengths, counts, t, window)
        b = lengths.shape[0]
        if sinks is not None:
            sinks = np.ascontiguousarray(sinks, np.float32)
            if sinks.shape != (self.query_heads,):
                raise ValueError(f"sinks must be [{self.query_heads}]")
        dev = []
        try:
            for a in (q, table, lengths, first, sinks,
                      np.zeros((t, self.query_heads, self.value_width), np.uint16),
                      np.full((t, self.query_heads), -np.inf, np.float32)):
                dev.append(None if a is None else self.ctx.upload(a))
            self.attend_device(dev[0], t, dev[1], table.shape[1], dev[2], b, dev[5], scale, dev[3], window, dev[4], dev[6])
            return {"out": dev[5].download(), "lse": dev[6].download()}
        finally:
            for d in dev:
                if d is not None:
                    d.free()

    def read(self, pages) -> dict:
        """{"k_codes" [n, heads, page, width / 2], "k_scales", and "v_codes", "v_scales"} of the pages named."""
        self._open()
        names = ("k_codes", "k_scales", "v_codes", "v_scales")[:4 if self.apart else 2]
        pages = [int(p) for p in pages]
        if any(not 0 <= p < self.pages for p in pages):
            raise ValueError(f"pages must be in [0, {self.pages})")
        out = {}
        for name, d in zip(names, self._owned):
            size = d.nbytes // self.pages
            out[name] = np.stack([self.ctx.download(d.ptr + p * size, d.shape[1:], np.uint8) for p in pages]) if pages \
                else np.zeros((0, *d.shape[1:]), np.uint8)
        return out


class CachedAttention:
    """An attention layer of the block-32 projections over a cache of its latents: of 64 heads of 512 values and one key
    head, the last 64 of them rotated. Opened by NativeProjections.open_cache, with which it closes (or earlier, by its
    close()). For x [T, 5120]:

      q = heads(wq_b(norm(wq_a(x)) q_norm)), normalized and rotated;  k = wkv(x), normalized with kv_norm and rotated, into
      the cache;  o = attention(q, cache), rotated back;  y = wo_b(wo_a(o)), wo_a by groups of eight heads."""

    HEADS, WIDTH, DIMS = 64, 512, 64

    def __init__(self, projections, pages: int, page: int, table, *, max_tokens: int, max_batch: int, q_norm=None,
                 kv_norm=None, sinks=None, scale: float = 512 ** -0.5, window: int = 0, eps: float = 1e-6):
        ctx, layout = projections.ctx, projections.layout
        group_rows, group_width = WO_A[0] // WO_A_GROUPS, WO_A[1]
        if projections.block != 32 or not projections.has_wo_a:
            raise ValueError("a cache needs block-32 projections with wo_a")
        if any(layout.get(n, (0, 0))[0] != rows for n, rows in (("wq_b", self.HEADS * self.WIDTH), ("wkv", self.WIDTH))) \
                or "wq_a" not in layout or "wo_b" not in layout or layout["wq_a"][0] != layout["wq_b"][1] \
                or layout["wq_a"][1] != layout["wkv"][1] or layout["wo_b"][1] != WO_A[0] \
                or self.HEADS * self.WIDTH != WO_A_GROUPS * group_width:
            raise ValueError("the projections are not of 64 heads over latents of 512")
        if not (math.isfinite(scale) and scale > 0) or window < 0:
            raise ValueError("scale must be positive and window not negative")
        if table is None or not 1 <= max_tokens <= MAX_TOKENS // self.HEADS:
            raise ValueError(f"a cache needs the rotation's table and max_tokens in [1, {MAX_TOKENS // self.HEADS}]")
        self.hidden, self.rank = layout["wq_a"][1], layout["wq_a"][0]
        weights = [None if w is None else np.ascontiguousarray(w, np.float32) for w in (q_norm, kv_norm, sinks)]
        for name, w, n in zip(("q_norm", "kv_norm", "sinks"), weights, (self.rank, self.WIDTH, self.HEADS)):
            if w is not None and w.shape != (n,):
                raise ValueError(f"{name} must be [{n}]")
        self.projections, self.ctx = projections, ctx
        self.scale, self.window, self.max_tokens = float(scale), int(window), int(max_tokens)
        self.lock, self._owned = threading.Lock(), []
        try:
            self.cache = self._own(KVCache4(ctx, pages, page, 1, self.WIDTH, self.WIDTH, query_heads=self.HEADS,
                                            max_tokens=max_tokens, max_batch=max_batch))
            self.down = self._own(HeadRotation(ctx, self.rank, norm=self.rank, eps=eps))
            self.heads = self._own(HeadRotation(ctx, self.WIDTH, norm=self.WIDTH, dims=self.DIMS, eps=eps, table=table))
            self.back = self._own(HeadRotation(ctx, self.WIDTH, dims=self.DIMS, table=table))
            self.q_norm, self.kv_norm, self.sinks = (None if w is None else self._own(ctx.upload(w)) for w in weights)
            for name in ("wq_a", "wq_b", "wkv", "wo_b"):   # so that a first step can be captured
                ctx.lib.fp8_reserve(ctx._h(), *layout[name], self.max_tokens)
            ctx.lib.fp8_reserve(ctx._h(), *WO_A, min(self.max_tokens, GROUPED_MAX_TOKENS))
            wide, tokens = self.HEADS * self.WIDTH, self.max_tokens
            self.qa, self.q, self.k, self.o, self.codes, self.scales, self.grouped = (
                self._own(ctx.empty((tokens, n), t)) for n, t in (
                    (self.rank, np.uint16), (wide, np.uint16), (self.WIDTH, np.uint16), (wide, np.uint16),
                    (wide, np.uint8), (wide // 32, np.uint8), (WO_A_GROUPS * group_rows, np.uint16)))
        except BaseException:
            self.close()
            raise

    def _own(self, thing):
        self._owned.append(thing)
        return thing

    def close(self):
        with self.lock:
            while self._owned:
                held = self._owned.pop()
                (held.close if hasattr(held, "close") else held.free)()

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def _open(self):
        if not self._owned:
            raise RuntimeError("the cache is closed")
        self.projections._ready()

    # -- device pointers in and out, no host synchronisation ---------------------------------------
    def step_device(self, x_ptr, tokens: int, positions_ptr, slots_ptr, table_ptr, columns: int, lengths_ptr, batch: int,
                    y_ptr, q_first_ptr=None, stream=None):
        """y [T, hidden] of x [T, hidden], both BF16: the tokens' latents go into device int64 slots [T] (outside the
        cache: not stored) at int32 positions [T], then each token attends to its sequence's `lengths` [batch] tokens on
        pages `table` [batch, columns], its own among them. The tokens are the last of their sequences: as many of each,
        or those that int32 q_first [batch + 1] gives. Rows of y behind the last sequence are of no use: what an earlier
        step left of its attention, projected. Threads take turns on one layer; device calls on the runtime beside it (another
        layer's step_device, project_device) share the context's scratch and are the caller's to order."""
        with self.lock:
            self._open()
            if not 0 <= tokens <= self.max_tokens or not 0 <= batch <= self.cache.max_batch:
                raise ValueError(f"the cache was opened for {self.max_tokens} tokens of {self.cache.max_batch} sequences a call")
            if not tokens:
                return
            # what the attention would refuse is refused before the tokens' latents are stored
            if q_first_ptr is None and (not batch or tokens % batch):
                raise ValueError("query rows do not divide among the sequences")
            if not 1 <= columns <= (1 << 30) // self.cache.page:
                raise ValueError(f"columns must be in [1, {(1 << 30) // self.cache.page}]")
            if batch and (not _lib.ptr(table_ptr) or not _lib.ptr(lengths_ptr) or _lib.ptr(table_ptr) % 4 or _lib.ptr(lengths_ptr) % 4
                          or (_lib.ptr(q_first_ptr) or 0) % 4):
                raise ValueError("table, lengths and q_first must be aligned device addresses")
            proj, lib, handle, vp = self.projections, self.ctx.lib, self.ctx._h(), _lib.vp
            rows, width = WO_A[0] // WO_A_GROUPS, WO_A[1]
            proj.project_device("wkv", x_ptr, tokens, self.k.ptr, stream)
            self.cache.append_device(self.k.ptr, slots_ptr, tokens, rotation=self.heads, positions_ptr=positions_ptr,
                                     weight_ptr=self.kv_norm, stream=stream)
            proj.project_device("wq_a", x_ptr, tokens, self.qa.ptr, stream)
            self.down.apply_device([self.down.set(self.qa, 1, self.qa, self.q_norm)], tokens, stream=stream)
            proj.project_device("wq_b", self.qa.ptr, tokens, self.q.ptr, stream)
            self.heads.apply_device([self.heads.set(self.q, self.HEADS, self.q)], tokens, positions_ptr, stream=stream)
            self.cache.attend_device(self.q, tokens, table_ptr, columns, lengths_ptr, batch, self.o, self.scale, q_first_ptr,
                                     self.window, self.sinks, stream=stream)
            self.back.apply_device([self.back.set(self.o, self.HEADS, self.o)], tokens, positions_ptr, inverse=True,
                                   stream=stream)
            lib.kv_round32(handle, vp(self.o), tokens * self.HEADS * self.WIDTH, vp(self.q), vp(self.codes), vp(self.scales),
                           _lib._stream(stream))   # (the rounded values take the queries' place)
            for t in range(0, tokens, GROUPED_MAX_TOKENS):
                lib.fp8_grouped_projection(handle, C.c_void_p(proj.tiled["wo_a"]), WO_A_GROUPS, rows, width,
                                           C.c_void_p(self.codes.ptr + t * WO_A_GROUPS * width),
                                           C.c_void_p(self.scales.ptr + t * WO_A_GROUPS * width // 32),
                                           min(GROUPED_MAX_TOKENS, tokens - t),
                                           C.c_void_p(self.grouped.ptr + t * WO_A_GROUPS * rows * 2), None, _lib._stream(stream))
            proj.project_device("wo_b", self.grouped.ptr, tokens, y_ptr, stream)

    # -- host arrays -------------------------------------------------------------------------------
    def step(self, x, positions, slots, table, lengths, counts=None) -> np.ndarray:
        """y [T, hidden] BF16 bits: x [T, hidden] BF16 bits, positions [T], slots [T], table [B, columns] and lengths [B]
        with the tokens of this step; counts [B] of them of each sequence (None: as many of each). Rows behind the last
        sequence are stored where they have a slot, and zero in y."""
        with self.projections.lock:
            self._open()
            t = validate_values(x, self.hidden)
            if x.ndim != 2 or t > self.max_tokens:
                raise ValueError(f"x must be [T, {self.hidden}] with T of at most {self.max_tokens}")
            positions = self.heads._positions(positions, t)
            slots = self.cache._slots(slots, t)
            table, lengths, first = self.cache._sequences(table, lengths, counts, t, self.window)
            dev = []
            try:
                for a in (x, positions, slots, table, lengths, first):
                    dev.append(None if a is None else self.ctx.upload(a))
                dev.append(self.ctx.empty((t, self.hidden), np.uint16))
                ptr = [None if d is None else d.ptr for d in dev]
                self.step_device(ptr[0], t, ptr[1], ptr[2], ptr[3], table.shape[1], ptr[4], lengths.shape[0], ptr[6], ptr[5])
                y = dev[6].download()
                if first is not None:
                    y[first[-1]:] = 0
                return y
            finally:
                for d in dev:
                    if d is not None:
                        d.free()
