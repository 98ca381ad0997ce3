"""Adapters of many requests beside one shared base model, over the C ABI (no
reference counterpart: the reference serves one model without adapters).

AdapterPlan says which adapter every row of a packed batch uses; LowRank adds
low-rank adapters next to a shared projection (runtime.Q8Weight); BlockNorm is
the norms after a block and before the next one with the block's gate and
residual scale. Device buffers are passed by address (e.g. a torch tensor's
data_ptr()); `stream` 0 is the context's stream.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from _lib import ABSMAX_ALL_ROWS, ABSMAX_PER_SEQUENCE
from _lib import DTYPE_BF16 as BF16
from _lib import DTYPE_F16 as F16
from _lib import DTYPE_F32 as F32
from _lib import Context, check, load


class _Handle:
    _free = ""

    def close(self) -> None:
        if getattr(self, "handle", None):
            getattr(load(), self._free)(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class AdapterPlan(_Handle):
    """sem_adapter_plan: batches of up to max_rows rows in up to max_seqs sequences."""
    _free = "sem_adapter_plan_free"

    def __init__(self, ctx: Context, max_rows: int, max_seqs: int):
        h = C.c_void_p()
        check(load().sem_adapter_plan_create(ctx.handle, max_rows, max_seqs, C.byref(h)))
        self.handle, self.ctx = h, ctx

    def set(self, offsets, adapters, stream: int = 0) -> None:
        """Rows [offsets[s], offsets[s+1]) use adapters[s] (-1: none)."""
        offsets = np.ascontiguousarray(offsets, dtype=np.int32)
        adapters = np.ascontiguousarray(adapters, dtype=np.int32)
        if offsets.ndim != 1 or adapters.ndim != 1 or offsets.size != adapters.size + 1:
            raise ValueError(f"adapter plan: {offsets.size} offsets for {adapters.size} sequences, want one more")
        check(load().sem_adapter_plan_set(self.handle, offsets.ctypes.data, adapters.ctypes.data, adapters.size,
                                          stream or None))


_NUMPY = {F32: np.float32, F16: np.float16, BF16: np.uint16}


def _weights(w, dtype: int, shape: tuple, what: str):
    """A contiguous array of `shape` in the bank's type (bf16 as its 16-bit patterns)."""
    w = np.asarray(w)
    if dtype == BF16 and w.dtype.itemsize == 2 and w.dtype.kind in "iu":
        w = w.view(np.uint16)
    if w.dtype != _NUMPY[dtype]:
        raise ValueError(f"{what}: {w.dtype} weights for a bank of type {dtype}")
    if w.shape != shape:
        raise ValueError(f"{what}: shape {w.shape}, want {shape}")
    return np.ascontiguousarray(w)


class LowRank(_Handle):
    """sem_lowrank: a[i] [rank][k_in] and b[i] [n_out][rank] numpy arrays of
    `dtype` (bf16 as int16 or uint16 bit patterns), both None for an adapter
    that leaves this projection as it is; scales[i] its factor."""
    _free = "sem_lowrank_free"

    def __init__(self, ctx: Context, k_in: int, n_out: int, a, b, scales, dtype: int = F16):
        if dtype not in _NUMPY:
            raise ValueError(f"low-rank adapters: unknown element type {dtype}")
        n = len(a)
        if len(b) != n or len(scales) != n:
            raise ValueError(f"low-rank adapters: {n} a, {len(b)} b and {len(scales)} scales")
        ranks = np.zeros(n, dtype=np.int32)
        keep, pa, pb = [], (C.c_void_p * max(n, 1))(), (C.c_void_p * max(n, 1))()
        for i in range(n):
            if a[i] is None and b[i] is None:
                continue
            if a[i] is None or b[i] is None:
                raise ValueError(f"low-rank adapter {i}: one of its two weights is missing")
            ranks[i] = r = np.shape(a[i])[0]
            wa = _weights(a[i], dtype, (r, k_in), f"low-rank adapter {i}: a")
            wb = _weights(b[i], dtype, (n_out, r), f"low-rank adapter {i}: b")
            keep += [wa, wb]
            pa[i], pb[i] = wa.ctypes.data, wb.ctypes.data
        s = np.ascontiguousarray(scales, dtype=np.float32)
        h = C.c_void_p()
        check(load().sem_lowrank_create(ctx.handle, k_in, n_out, n, ranks.ctypes.data, s.ctypes.data, pa, pb, dtype,
                                        C.byref(h)))
        self.handle, self.ctx, self.k_in, self.n_out, self.ranks = h, ctx, k_in, n_out, ranks

    def apply(self, plan: AdapterPlan, d_x: int, x_dtype: int, d_y: int, y_dtype: int, d_base: int = 0, ldx: int = 0,
              ld_base: int = 0, ldy: int = 0, stream: int = 0) -> None:
        """y = base + scale * (x a^T) b^T for every row of the plan's batch
        (d_base 0: no base; it may be d_y)."""
        check(load().sem_lowrank_apply(self.handle, plan.handle, d_x, x_dtype, ldx, d_base or None, ld_base, d_y,
                                       y_dtype, ldy, stream or None))

    def apply_int8(self, plan: AdapterPlan, d_codes: int, d_absmax: int, n_absmax: int, d_y: int, d_base: int = 0,
                   ld_base: int = 0, ldy: int = 0, stream: int = 0) -> None:
        """The same on INT8 codes held as fp16 with one activation scale (n_absmax 1 or ABSMAX_ALL_ROWS), or one per
        sequence (their number or ABSMAX_PER_SEQUENCE; by name in a capture on a plan of one sequence)."""
        check(load().sem_lowrank_apply_int8(self.handle, plan.handle, d_codes, d_absmax, n_absmax, d_base or None,
                                            ld_base, d_y, ldy, stream or None))

    def check(self) -> None:
        """Waits for the device and raises what the calls recorded (sem_lowrank_check)."""
        check(load().sem_lowrank_check(self.handle))


class BlockNorm(_Handle):
    """sem_block_norm: post and pre weights [dim] (None: that norm is left
    out), gates [n][dim] and scales [n] of the adapters (None: 1)."""
    _free = "sem_block_norm_free"

    def __init__(self, ctx: Context, dim: int, eps: float, post=None, pre=None, gates=None, scales=None):
        def vector(w, shape, what):
            if w is None:
                return None
            w = np.ascontiguousarray(w, dtype=np.float32)
            if w.shape != shape:
                raise ValueError(f"block norm: {what} of shape {w.shape}, want {shape}")
            return w

        n = len(gates) if gates is not None else len(scales) if scales is not None else 0
        post, pre = vector(post, (dim,), "post"), vector(pre, (dim,), "pre")
        gates, scales = vector(gates, (n, dim), "gates"), vector(scales, (n,), "scales")
        address = lambda w: w.ctypes.data if w is not None and w.size else None  # noqa: E731
        h = C.c_void_p()
        check(load().sem_block_norm_create(ctx.handle, dim, eps, address(post), address(pre), n, address(gates),
                                           address(scales), C.byref(h)))
        self.handle, self.ctx, self.dim, self.n_adapters = h, ctx, dim, n

    def run(self, rows: int, d_o: int, dtype: int, d_h: int, h_dtype: int, d_h_out: int, d_y: int = 0,
            plan: AdapterPlan | None = None, ldo: int = 0, ldh: int = 0, ld_h_out: int = 0, ldy: int = 0,
            stream: int = 0) -> None:
        """h_out = scale * h + gate * rmsnorm(o) * post; y = rmsnorm(h_out) * pre."""
        check(load().sem_block_norm_run(self.handle, plan.handle if plan is not None else None, rows, d_o, ldo, dtype,
                                        d_h, ldh, h_dtype, d_h_out, ld_h_out, d_y or None, ldy, stream or None))


__all__ = ["AdapterPlan", "LowRank", "BlockNorm", "F32", "F16", "BF16", "ABSMAX_ALL_ROWS", "ABSMAX_PER_SEQUENCE"]
