"""Tokens sorted by expert and back, on the device, with their gradients.

ExpertDispatch is the batched, device-side form of participation and MoEAccumulator (src/vesper/moe.py:18-148) for
experts of any format: `dispatch` builds the plan of a routing table (rows ordered by expert, ascending tokens within
one) and moves the tokens' rows into that order, the experts run on their slices of it, and `combine` adds each token's
rows in ascending expert order, the shared expert's row last, with one rounding. `combine_backward` and
`dispatch_backward` are their gradients.

An id outside [0, experts) names an expert of another device: its pair gets no row, adds nothing and has zero gradient.

The *_device methods take device pointers and do not synchronise; dispatch, combine and the backward methods take and
return host arrays (BF16 as uint16 bits, or FP32). The plan of the latest dispatch stays in the object's buffers, so
calls on one object must not overlap on different streams; a plan that has to outlive the next dispatch (two
micro-batches in flight) takes an object of its own.
"""

from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib

MAX_TOKENS, MAX_TOP_K, MAX_EXPERTS, MAX_WIDTH = 1 << 18, 32, 1024, 1 << 24
_HOST_TYPES = {np.dtype(np.uint16): "bf16", np.dtype(np.float32): "f32", np.dtype(np.uint8): "u8"}


def row_type(name: str, bytes_too: bool = False) -> int:
    if name not in _lib.MX_ROWS or (name == "u8" and not bytes_too):
        raise ValueError(f"row type must be {'bf16, f32 or u8' if bytes_too else 'bf16 or f32'}")
    return _lib.MX_ROWS[name]


def host_rows(array, rows: int | None = None, bytes_too: bool = False):
    """(contiguous array, row type) of a host [rows, width] array: uint16 BF16 bits, FP32, or bytes where they move."""
    array = np.asarray(array)
    name = _HOST_TYPES.get(array.dtype)
    if name is None or (name == "u8" and not bytes_too) or array.ndim != 2:
        raise ValueError("rows must be a 2-D array of BF16 storage bits (uint16) or FP32 values")
    if rows is not None and array.shape[0] != rows:
        raise ValueError(f"expected {rows} rows, got {array.shape[0]}")
    if not 1 <= array.shape[1] <= MAX_WIDTH:
        raise ValueError(f"row width outside [1, {MAX_WIDTH}]")
    return np.ascontiguousarray(array), name


class RowPlan(_lib.MxRowPlan):
    """The device addresses of an ExpertDispatch's plan, and the object that knows what it was made for."""

    def __init__(self, dispatch: ExpertDispatch):
        super().__init__(dispatch.first, dispatch.pair_row, dispatch.row_pair)
        self.dispatch = dispatch


class ExpertDispatch:
    def __init__(self, ctx: _lib.Context, experts: int, top_k: int, max_tokens: int):
        if not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= MAX_TOP_K or not 1 <= max_tokens <= MAX_TOKENS:
            raise ValueError(f"experts in [1, {MAX_EXPERTS}], top_k in [1, {MAX_TOP_K}] and max_tokens in "
                             f"[1, {MAX_TOKENS}] required")
        self.ctx, self.experts, self.top_k, self.max_tokens = ctx, int(experts), int(top_k), int(max_tokens)
        pairs = self.max_tokens * self.top_k
        self._owned = []
        try:
            for count in (self.experts + 1, pairs, pairs):
                self._owned.append(ctx.empty((count,), np.int32))
        except BaseException:
            self.close()
            raise
        self.first, self.pair_row, self.row_pair = (d.ptr for d in self._owned)
        self.tokens = None   # of the plan in the buffers
        self.plan = RowPlan(self)

    def close(self):
        for d in self._owned:
            d.free()
        self._owned.clear()

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def _open(self, tokens=None) -> int:
        if not self._owned:
            raise RuntimeError("the dispatch is closed")
        if tokens is None:
            if self.tokens is None:
                raise RuntimeError("no routing has been dispatched")
            return self.tokens
        if not 0 <= int(tokens) <= self.max_tokens:
            raise ValueError(f"token count outside [0, {self.max_tokens}]")
        return int(tokens)

    # -- device pointers in and out, no host synchronisation ---------------------------------------
    def plan_device(self, ids_ptr, tokens: int, stream=None):
        """The plan of ids [tokens, top_k] (device int32) alone."""
        t = self._open(tokens)
        self.ctx.lib.dispatch(self.ctx._h(), _lib.vp(ids_ptr), t, self.top_k, self.experts, C.byref(self.plan), None,
                              0, 0, None, None, None, _lib._stream(stream))
        self.tokens = t

    def dispatch_device(self, ids_ptr, tokens: int, x_ptr, width: int, rows_ptr, dtype: str = "bf16",
                        weights_ptr=None, row_weights_ptr=None, stream=None):
        """The plan of ids, and x [tokens, width] as rows [tokens * top_k, width] in expert order, with the route
        weights in the same order where they are given."""
        t, code = self._open(tokens), row_type(dtype, True)
        self.ctx.lib.dispatch(self.ctx._h(), _lib.vp(ids_ptr), t, self.top_k, self.experts, C.byref(self.plan),
                              _lib.vp(x_ptr), code, int(width), _lib.vp(weights_ptr),
                              _lib.vp(rows_ptr), _lib.vp(row_weights_ptr), _lib._stream(stream))
        self.tokens = t

    def move_device(self, x_ptr, width: int, rows_ptr, dtype: str = "bf16", stream=None):
        """A further tensor of the dispatched tokens (block scales beside codes) by the present plan."""
        t, code = self._open(), row_type(dtype, True)
        self.ctx.lib.dispatch(self.ctx._h(), None, t, self.top_k, self.experts, C.byref(self.plan), _lib.vp(x_ptr),
                              code, int(width), None, _lib.vp(rows_ptr), None, _lib._stream(stream))

    def combine_device(self, rows_ptr, width: int, y_ptr, dtype: str = "bf16", weights_ptr=None, shared_ptr=None,
                       stream=None):
        t, code = self._open(), row_type(dtype)
        self.ctx.lib.combine(self.ctx._h(), _lib.vp(rows_ptr), code, C.c_void_p(self.pair_row),
                             _lib.vp(weights_ptr), _lib.vp(shared_ptr), t, self.top_k, int(width), _lib.vp(y_ptr),
                             _lib._stream(stream))

    def combine_backward_device(self, dy_ptr, rows_ptr, width: int, drows_ptr, dweights_ptr=None, dtype: str = "bf16",
                                weights_ptr=None, stream=None):
        t, code = self._open(), row_type(dtype)
        self.ctx.lib.combine_backward(self.ctx._h(), _lib.vp(dy_ptr), _lib.vp(rows_ptr), code,
                                      C.c_void_p(self.pair_row), _lib.vp(weights_ptr), t, self.top_k, int(width),
                                      _lib.vp(drows_ptr), _lib.vp(dweights_ptr), _lib._stream(stream))

    def dispatch_backward_device(self, drows_ptr, width: int, dx_ptr, dtype: str = "bf16", drow_weights_ptr=None,
                                 dweights_ptr=None, stream=None):
        t, code = self._open(), row_type(dtype)
        self.ctx.lib.dispatch_backward(self.ctx._h(), _lib.vp(drows_ptr), code, C.c_void_p(self.pair_row),
                                       _lib.vp(drow_weights_ptr), t, self.top_k, int(width), _lib.vp(dx_ptr),
                                       _lib.vp(dweights_ptr), _lib._stream(stream))

    # -- host arrays -------------------------------------------------------------------------------
    def _ids(self, ids) -> np.ndarray:
        ids = np.asarray(ids)
        if ids.dtype not in (np.dtype(np.int32), np.dtype(np.int64)) or ids.ndim != 2 or ids.shape[1] != self.top_k:
            raise ValueError(f"routing must be an integer array [T, {self.top_k}]")
        if ids.size and (ids.min() < -2 ** 31 or ids.max() >= 2 ** 31):
            raise ValueError("routing ids must fit 32 bits")
        self._open(ids.shape[0])
        return np.ascontiguousarray(ids, np.int32)

    def _pair_values(self, values, tokens, what) -> np.ndarray | None:
        if values is None:
            return None
        values = np.ascontiguousarray(values, np.float32)
        if values.shape != (tokens, self.top_k):
            raise ValueError(f"{what} must be [{tokens}, {self.top_k}]")
        return values

    def _call(self, inputs, outputs, method):
        """`method(*device arrays)` on uploaded inputs (None stays None) and zeroed outputs [(shape, dtype)]; the
        outputs as host arrays."""
        dev = []
        try:
            for a in inputs:
                dev.append(None if a is None else self.ctx.upload(a))
            for shape, dtype in outputs:
                dev.append(self.ctx.upload(np.zeros(shape, dtype)))
            method(*dev)
            return [d.download() for d in dev[len(inputs):]]
        finally:
            for d in dev:
                if d is not None:
                    d.free()

    def read_plan(self) -> dict:
        """{"first" [experts + 1], "pair_row" [T, k], "row_pair" [T k]} of the present plan."""
        pairs = self._open() * self.top_k
        return {"first": self.ctx.download(self.first, (self.experts + 1,), np.int32),
                "pair_row": self.ctx.download(self.pair_row, (self.tokens, self.top_k), np.int32),
                "row_pair": self.ctx.download(self.row_pair, (pairs,), np.int32)}

    def dispatch(self, ids, x, weights=None) -> dict:
        """ids [T, k] and x [T, width] -> the plan (read_plan), "rows" [T k, width] (zero from first[experts] on) and,
        with weights [T, k], "row_weights" [T k]."""
        ids = self._ids(ids)
        t, pairs = ids.shape[0], ids.size
        x, dtype = host_rows(x, t, bytes_too=True)
        weights = self._pair_values(weights, t, "route weights")
        outputs = [((pairs, x.shape[1]), x.dtype)] + ([] if weights is None else [((pairs,), np.float32)])

        def call(ids_d, x_d, w_d, rows_d, row_weights_d=None):
            self.dispatch_device(ids_d, t, x_d, x.shape[1], rows_d, dtype, w_d, row_weights_d)
        moved = self._call([ids, x, weights], outputs, call)
        return dict(self.read_plan(), rows=moved[0], **({} if weights is None else {"row_weights": moved[1]}))

    def combine(self, rows, weights=None, shared=None) -> np.ndarray:
        """[T, width] of the rows [T k, width] of the dispatched tokens' experts, in the rows' type."""
        t = self._open()
        rows, dtype = host_rows(rows, t * self.top_k)
        weights = self._pair_values(weights, t, "route weights")
        if shared is not None:
            shared, shared_type = host_rows(shared, t)
            if shared_type != dtype or shared.shape[1] != rows.shape[1]:
                raise ValueError("the shared expert's rows must have the type and width of the experts' rows")
        return self._call([rows, weights, shared], [((t, rows.shape[1]), rows.dtype)],
                          lambda r, w, s, y: self.combine_device(r, rows.shape[1], y, dtype, w, s))[0]

    def combine_backward(self, dy, rows, weights=None) -> dict:
        """{"drows" [T k, width], "dweights" [T, k]} for dy [T, width]; the gradient of `shared` is dy."""
        t = self._open()
        dy, dtype = host_rows(dy, t)
        rows, rows_dtype = host_rows(rows, t * self.top_k)
        if rows_dtype != dtype or rows.shape[1] != dy.shape[1]:
            raise ValueError("rows and their gradient must have one type and width")
        weights = self._pair_values(weights, t, "route weights")
        out = self._call([dy, rows, weights], [(rows.shape, rows.dtype), ((t, self.top_k), np.float32)],
                         lambda g, r, w, dr, dw: self.combine_backward_device(g, r, rows.shape[1], dr, dw, dtype, w))
        return {"drows": out[0], "dweights": out[1]}

    def dispatch_backward(self, drows, drow_weights=None) -> dict:
        """{"dx" [T, width]} for drows [T k, width], and "dweights" [T, k] for drow_weights [T k]."""
        t = self._open()
        drows, dtype = host_rows(drows, t * self.top_k)
        outputs = [((t, drows.shape[1]), drows.dtype)]
        if drow_weights is not None:
            drow_weights = np.ascontiguousarray(drow_weights, np.float32)
            if drow_weights.shape != (t * self.top_k,):
                raise ValueError(f"drow_weights must be [{t * self.top_k}]")
            outputs.append(((t, self.top_k), np.float32))

        def call(dr, dw_rows, dx, dw=None):
            self.dispatch_backward_device(dr, drows.shape[1], dx, dtype, dw_rows, dw)
        out = self._call([drows, drow_weights], outputs, call)
        return dict(zip(("dx", "dweights"), out))
