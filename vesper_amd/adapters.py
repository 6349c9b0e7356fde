"""Low-rank adapters of many requests beside a projection (no counterpart in the reference, whose projections are
fixed: src/vesper/projections.py).

AdapterBank keeps `slots` adapters of one projection of `rows` by `width` resident: down [rank, width] and up
[rows, rank] (BF16) with a scale, each of a rank of its own up to `max_rank`. One call gives every token the adapter of
its request: y[t] = base[t] + scale up (down x[t]) with slot ids[t], and y[t] = base[t] where ids[t] names no loaded
slot. `base` is the projection's BF16 output or, for a single rounding, its FP32 sums (the trace). NativeProjections
opens banks beside its own matrices (open_adapters) and applies them in fp8().

The bank has one workspace: calls on one bank must not overlap on different streams.
"""

from __future__ import annotations

import ctypes as C
import math

import numpy as np

from . import _lib
from .dispatch import ExpertDispatch, RowPlan

MAX_SLOTS, MAX_RANK, MAX_TOKENS, MAX_SIZE = 1024, 256, 1 << 18, 1 << 20


def _bf16(array, shape, what) -> np.ndarray:
    array = np.asarray(array)
    if array.dtype != np.uint16 or array.shape != shape or np.any((array & 0x7F80) == 0x7F80):
        raise ValueError(f"{what} must be finite BF16 storage bits of shape {shape}")
    return np.ascontiguousarray(array)


class AdapterBank:
    def __init__(self, ctx: _lib.Context, rows: int, width: int, slots: int, max_rank: int, max_tokens: int):
        if min(rows, width) < 8 or rows % 8 or width % 8 or max(rows, width) > MAX_SIZE:
            raise ValueError(f"rows and width must be multiples of 8 in [8, {MAX_SIZE}]")
        if not 1 <= slots <= MAX_SLOTS or not 1 <= max_rank <= MAX_RANK or not 1 <= max_tokens <= MAX_TOKENS:
            raise ValueError(f"slots in [1, {MAX_SLOTS}], max_rank in [1, {MAX_RANK}] and max_tokens in "
                             f"[1, {MAX_TOKENS}] required")
        self.ctx, self.rows, self.width = ctx, int(rows), int(width)
        self.slots, self.max_rank, self.max_tokens = int(slots), int(max_rank), int(max_tokens)
        self.few_tokens = 128 if self.max_rank <= 64 else 64   # calls of up to so many find each adapter's tokens anew
        handle = C.c_void_p()
        ctx.lib.adapters_create(ctx._h(), self.rows, self.width, self.slots, self.max_rank, C.byref(handle))
        self.handle, self.workspace = handle, 0
        try:
            self.workspace_bytes = int(ctx.lib.cdll.mx_adapters_workspace_bytes(handle, self.max_tokens))
            self.workspace = ctx.malloc(self.workspace_bytes)
        except BaseException:
            self.close()
            raise

    def close(self):
        if self.handle:
            self.ctx._h()   # a closed context has taken the bank with it
            handle, self.handle = self.handle, C.c_void_p()
            self.ctx.lib.adapters_destroy(handle)
        if self.workspace:
            workspace, self.workspace = self.workspace, 0
            self.ctx.free(workspace)

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def _open(self):
        if not self.handle:
            raise RuntimeError("the adapter bank is closed")
        self.ctx._h()

    def _slot(self, slot, rank, scale):
        self._open()
        if type(slot) is not int or not 0 <= slot < self.slots:
            raise ValueError(f"slot outside [0, {self.slots})")
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"adapter rank outside [1, {self.max_rank}]")
        if not math.isfinite(C.c_float(scale).value):
            raise ValueError("adapter scale must be a finite FP32 value")

    # -- loading ----------------------------------------------------------------------------------
    def load_device(self, slot: int, down_ptr, up_ptr, rank: int, scale: float = 1.0, stream=None):
        """Slot <- device BF16 down [rank, width] and up [rows, rank], ordered on `stream`. The weights must be finite
        (load checks it)."""
        self._slot(slot, rank, scale)
        self.ctx.lib.adapters_load(self.handle, slot, _lib.vp(down_ptr), _lib.vp(up_ptr), int(rank), float(scale),
                                   _lib._stream(stream))

    def load(self, slot: int, down, up, scale: float = 1.0):
        """Slot <- host BF16 bits (uint16) down [rank, width] and up [rows, rank]."""
        rank = np.asarray(down).shape[0] if np.ndim(down) == 2 else 0
        self._slot(slot, rank, scale)
        down, up = _bf16(down, (rank, self.width), "down"), _bf16(up, (self.rows, rank), "up")
        dev = []
        try:
            for a in (down, up):
                dev.append(self.ctx.upload(a))
            self.load_device(slot, dev[0], dev[1], rank, scale)
            self.ctx.sync()
        finally:
            for d in dev:
                d.free()

    def clear(self, slot: int, stream=None):
        """Empty the slot: tokens that name it get their base."""
        self._slot(slot, 1, 1.0)
        self.ctx.lib.adapters_load(self.handle, slot, None, None, 0, 0.0, _lib._stream(stream))

    # -- calls ------------------------------------------------------------------------------------
    def apply_device(self, x_ptr, ids_ptr, tokens: int, base_ptr, y_ptr, base_dtype: str = "bf16", x_stride=None,
                     base_stride=None, y_stride=None, plan=None, stream=None):
        """y [tokens, rows] BF16 of x [tokens, width] BF16, base [tokens, rows] and int32 ids [tokens]; strides in
        values (None: contiguous). plan: ExpertDispatch(ctx, slots, 1, tokens) after plan_device(ids, tokens), or its
        .plan, made once for all projections of a step whose banks have as many slots; None makes it within the call,
        and up to few_tokens no plan is read. (An MxRowPlan of a caller's own is taken as it is.) No synchronisation."""
        self._open()
        if not 0 <= tokens <= self.max_tokens:
            raise ValueError(f"token count outside [0, {self.max_tokens}]")
        if base_dtype not in ("bf16", "f32"):
            raise ValueError("base type must be bf16 or f32")
        plan = self.check_plan(plan, tokens)
        ptr = _lib.ptr
        x_stride = self.width if x_stride is None else x_stride
        base_stride = self.rows if base_stride is None else base_stride
        y_stride = self.rows if y_stride is None else y_stride
        self.ctx.lib.adapters_apply(self.handle, ptr(x_ptr), x_stride, ptr(ids_ptr),
                                    None if plan is None else C.byref(plan), tokens, ptr(base_ptr),
                                    _lib.MX_ROWS[base_dtype], base_stride, ptr(y_ptr), y_stride, self.workspace,
                                    self.workspace_bytes, None if stream is None else int(stream))

    def check_plan(self, plan, tokens: int) -> _lib.MxRowPlan | None:
        """The plan that a call of `tokens` tokens reads, None if it reads none."""
        if plan is None:
            return None
        if not isinstance(plan, (ExpertDispatch, _lib.MxRowPlan)):
            raise TypeError("plan must be an ExpertDispatch or its plan")
        if tokens <= self.few_tokens:
            return None
        if isinstance(plan, RowPlan):
            plan = plan.dispatch
        if not isinstance(plan, ExpertDispatch):
            return plan
        made = plan._open()
        if (plan.experts, plan.top_k, made, plan.ctx.ordinal) != (self.slots, 1, tokens, self.ctx.ordinal):
            raise ValueError(f"the plan is of {made} tokens with {plan.top_k} of {plan.experts} groups on device "
                             f"{plan.ctx.ordinal}; this call takes {tokens} with 1 of {self.slots} on {self.ctx.ordinal}")
        return plan.plan

    def check_ids(self, ids, tokens: int) -> np.ndarray:
        """Host slot ids [tokens] as int32: each a slot of the bank, or -1 for none."""
        ids = np.asarray(ids)
        if ids.dtype not in (np.dtype(np.int32), np.dtype(np.int64)) or ids.shape != (tokens,):
            raise ValueError(f"adapter ids must be an integer array [{tokens}]")
        if ids.size and (ids.min() < -1 or ids.max() >= self.slots):
            raise ValueError(f"adapter ids must be in [-1, {self.slots})")
        return np.ascontiguousarray(ids, np.int32)

    def apply(self, x, ids, base) -> np.ndarray:
        """Host arrays: x [T, width] BF16 bits, ids [T], base [T, rows] BF16 bits or FP32 -> BF16 bits [T, rows]."""
        self._open()
        if np.ndim(x) != 2 or not 0 <= len(x) <= self.max_tokens:
            raise ValueError(f"x must be [T, {self.width}] with T in [0, {self.max_tokens}]")
        t = len(x)
        x, ids, base = _bf16(x, (t, self.width), "x"), self.check_ids(ids, t), np.asarray(base)
        if base.dtype not in (np.dtype(np.uint16), np.dtype(np.float32)) or base.shape != (t, self.rows):
            raise ValueError(f"base must be BF16 storage bits or FP32 values of shape ({t}, {self.rows})")
        dev = []
        try:
            for a in (x, ids, base, np.zeros((t, self.rows), np.uint16)):
                dev.append(self.ctx.upload(a))
            self.apply_device(dev[0], dev[1], t, dev[2], dev[3], "f32" if base.dtype == np.float32 else "bf16")
            return dev[3].download()
        finally:
            for d in dev:
                d.free()
