"""The 8-bit path over the C-ABI of include/ar_i8.h: rows in 8 bits with a scale each, the calls that make them from
floats (alone, or as the residual's norm), read them back, and multiply them.

No counterpart in the reference (its contexts compute in FP32 or FP64).  A feed-forward block:

    ops = Int8Ops(ctx)
    gate, up, down = (ops.rows(F, dim), ops.rows(F, dim), ops.rows(dim, F))  # weights, by output channel
    ops.quantize(w_gate, gate, DTYPE_BF16)                                   # once; up and down alike
    x8, act8 = ops.rows(tokens, dim), ops.rows(tokens, F)
    ops.add_rmsnorm_i8(h, norm_w, eps, x8, x=attn)                           # h += attn; x8 = rmsnorm(h)
    ops.gemm(x8, gate, act, epilogue=GEMM_SWIGLU, W2=up)                     # act = up * silu(gate)
    ops.quantize(act, act8)
    ops.gemm(act8, down, h, epilogue=GEMM_RESIDUAL)                          # h += down

Buffers are anything with a ``ptr`` (``hardware.DeviceBuffer``).  Everything runs on the context's stream.  Rows of another
context on the same device may be used (the order between the two streams is the caller's), of another device not.  A product
that needs more work space than any before it allocates it; the space that queued calls still use stays until ``close``.
"""
from __future__ import annotations

import ctypes
import weakref

from .hardware import DTYPE_F32, GEMM_STORE, HipContext, check, lib

KEPT_SIZES = 64  # work sizes that are kept


class ArRowsI8(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("stride", ctypes.c_int64),
                ("rows", ctypes.c_int32), ("n", ctypes.c_int32)]


def _ptr(buf):
    return buf.ptr if buf is not None else None


class Int8Rows:
    """`rows` rows of `n` values in 8 bits (ar_rows_i8): value (r, i) is q[r][i] * scale[r].  Buffers that are not given
    are allocated; given ones (q: `stride` bytes a row, a multiple of 16) stay the caller's."""

    def __init__(self, ctx: HipContext, rows: int, n: int, q=None, scale=None, stride: int = 0):
        self.ctx, self.rows, self.n = ctx, rows, n
        self.stride = stride or -(-n // 16) * 16
        self._own, self._parts = [], weakref.WeakSet()
        try:
            self.q = q if q is not None else self._take(rows * self.stride)
            self.scale = scale if scale is not None else self._take(rows * 4)
        except Exception:
            self.close()
            raise
        self._set()

    def _take(self, nbytes):
        buf = self.ctx.allocate(max(nbytes, 16))
        self._own.append(buf)
        return buf

    def _set(self):
        self.raw = ArRowsI8(_ptr(self.q), _ptr(self.scale), self.stride, self.rows, self.n)
        self.ref = ctypes.byref(self.raw)

    def first(self, rows: int) -> "Int8Rows":
        """The first `rows` rows, on the same buffers; they end with these."""
        if not 0 <= rows <= self.rows:
            raise ValueError(f"{rows} of {self.rows} rows")
        if self.q is None:
            raise ValueError("the rows are closed")
        part = Int8Rows(self.ctx, rows, self.n, self.q, self.scale, self.stride)
        self._parts.add(part)
        return part

    def close(self):
        """Frees the buffers these rows allocated; calls with them, or with rows taken from them, are refused after it."""
        for part in list(self._parts):
            part.close()
        for buf in self._own:
            buf.free()
        self._own = []
        self.q = self.scale = None
        self.raw = ArRowsI8(None, None, self.stride, self.rows, self.n)
        self.ref = ctypes.byref(self.raw)


class Int8Ops:
    """The 8-bit operators of a context, and the work space of their products."""

    def __init__(self, ctx: HipContext):
        self.ctx = ctx
        L = lib()  # (bound once: a decode step makes some hundred of these calls)
        self._quantize, self._embed = L.ar_hip_quantize_i8, L.ar_hip_embed_i8
        self._norm, self._norm_i8, self._gemm = L.ar_hip_add_rmsnorm, L.ar_hip_add_rmsnorm_i8, L.ar_hip_gemm_i8
        self._work, self._need = [], {}  # (_work: the last is in use; _need: work bytes by sizes)

    def close(self):
        for buf in self._work:
            buf.free()
        self._work = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _check_device(self, rows: Int8Rows):
        if rows.ctx not in (None, self.ctx) and rows.ctx.index != self.ctx.index:  # (None: on buffers of the caller's)
            raise ValueError(f"rows of device {rows.ctx.index} cannot be used on device {self.ctx.index}")

    def rows(self, rows: int, n: int) -> Int8Rows:
        """New rows in 8 bits."""
        return Int8Rows(self.ctx, rows, n)

    def quantize(self, x, out: Int8Rows, x_dtype: int = DTYPE_F32, x_stride: int = 0):
        """Rows of floats to 8 bits (ar_hip_quantize_i8).  A stride of 0, here and below: rows one after another."""
        self._check_device(out)
        rc = self._quantize(self.ctx.handle, _ptr(x), x_dtype, x_stride or out.n, out.ref)
        if rc:
            check(rc)

    def add_rmsnorm(self, h, w, eps: float, rows: int, n: int, y, x=None, h_dtype: int = DTYPE_F32,
                    x_dtype: int = DTYPE_F32, y_dtype: int = DTYPE_F32, h_stride: int = 0, x_stride: int = 0,
                    y_stride: int = 0):
        """h += x, y = rmsnorm(h) * w (ar_hip_add_rmsnorm)."""
        rc = self._norm(self.ctx.handle, _ptr(h), h_dtype, h_stride or n, _ptr(x), x_dtype, x_stride or n, _ptr(w), eps,
                        rows, n, _ptr(y), y_dtype, y_stride or n)
        if rc:
            check(rc)

    def add_rmsnorm_i8(self, h, w, eps: float, out: Int8Rows, x=None, h_dtype: int = DTYPE_F32,
                       x_dtype: int = DTYPE_F32, h_stride: int = 0, x_stride: int = 0):
        """h += x, out = rmsnorm(h) * w in 8 bits (ar_hip_add_rmsnorm_i8)."""
        self._check_device(out)
        rc = self._norm_i8(self.ctx.handle, _ptr(h), h_dtype, h_stride or out.n, _ptr(x), x_dtype, x_stride or out.n, _ptr(w),
                           eps, out.ref)
        if rc:
            check(rc)

    def embed(self, table: Int8Rows, tokens, count: int, y, y_dtype: int = DTYPE_F32, y_stride: int = 0):
        """Rows of the table by token (None: the first `count`) as floats (ar_hip_embed_i8)."""
        self._check_device(table)
        rc = self._embed(self.ctx.handle, table.ref, _ptr(tokens), count, _ptr(y), y_dtype, y_stride or table.n)
        if rc:
            check(rc)

    def _scratch(self, M, N, K, epilogue):
        need = self._need.get((M, N, K, epilogue))
        if need is None:
            b = ctypes.c_size_t()
            check(lib().ar_hip_gemm_i8_work(self.ctx.handle, M, N, K, epilogue, ctypes.byref(b)))
            need = b.value
            if len(self._need) >= KEPT_SIZES:  # (a server's row counts differ from step to step)
                self._need.clear()
            self._need[M, N, K, epilogue] = need
        if not need:
            return None
        work = self._work[-1] if self._work else None
        if work is None or work.nbytes < need:
            work = self.ctx.allocate(max(need, 2 * work.nbytes if work else 0))
            self._work.append(work)
        return work

    def gemm(self, A: Int8Rows, W: Int8Rows, C, epilogue: int = GEMM_STORE, W2: Int8Rows | None = None, bias=None,
             c_dtype: int = DTYPE_F32, ldc: int = 0):
        """C = A W^T, C += A W^T or C = (A W2^T) * silu(A W^T) of rows in 8 bits (ar_hip_gemm_i8)."""
        self._check_device(A)
        self._check_device(W)
        if W2 is not None:
            self._check_device(W2)
        w = self._scratch(A.rows, W.rows, A.n, epilogue)
        rc = self._gemm(self.ctx.handle, A.ref, W.ref, W2.ref if W2 is not None else None, _ptr(bias), _ptr(C), c_dtype,
                        ldc or W.rows, epilogue, _ptr(w), w.nbytes if w else 0)
        if rc:
            check(rc)
