"""Paged KV cache over the C-ABI of include/ar_pages.h: pools of pages that many sequences share, the calls that
take, share, give back and move pages, the row preparation and the attention of new tokens.

No counterpart in the reference (one contiguous cache per model, AttentionFeatures.java:823-826).  A token loop:

    cache = PagedCache(ctx, layers=28, pages=4096, kv_heads=8, head_size=128, seqs=16, max_pages=128)
    rows = Chunks(n, total, start=start, at=at)        # device int32 buffers; cache.grow fills `at`
    cache.grow(rows, missing)
    for layer in ...:
        ...                                            # projections: HipContext.gemm_f32 / gemm_bf16 / dense
        cache.write(layer, rows, q, k, v, q_out, heads, rotary)
        cache.attention(layer, rows, q_out, out, heads)

Buffers are anything with a ``ptr`` (``hardware.DeviceBuffer``).  Everything runs on the context's stream.  A call that
needs more work space than any before it allocates it; the space that queued calls still use stays until ``close``.
"""
from __future__ import annotations

import ctypes

import numpy as np

from .hardware import DTYPE_BF16, DTYPE_F16, DTYPE_F32, HipContext, check, lib

ROPE_SECTIONS, ROPE_INTERLEAVED = 0, 1
KEPT_SIZES = 64  # work sizes that a cache keeps
ELEM_BYTES = {DTYPE_F32: 4, DTYPE_BF16: 2, DTYPE_F16: 2}


class ArPages(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "table", "rows", "refs")] + \
               [(n, ctypes.c_int32) for n in ("dtype", "layers", "pages", "kv_heads", "page_rows", "head_dim", "seqs",
                                              "max_pages")]


class ArChunks(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("seq", "start", "at")] + [(n, ctypes.c_int32) for n in ("n", "rows")]


class ArRotary(ctypes.Structure):
    _fields_ = [("theta", ctypes.c_double), ("positions", ctypes.c_void_p), ("axes", ctypes.c_int32),
                ("layout", ctypes.c_int32), ("section", ctypes.c_int32 * 4)]


def _ptr(buf):
    return buf.ptr if buf is not None else None


class Chunks:
    """The new rows of a call by sequence (ar_chunks): `n` chunks, `rows` rows in the call's arrays; device int32
    buffers `start` [n+1] (None: one row each), `at` [n] (cache row of each chunk's first row) and `seq` [n] (None:
    sequences 0..n-1).  Holds its buffers."""

    def __init__(self, n: int, rows: int, at, start=None, seq=None):
        self.n, self.rows, self.at, self.start, self.seq = n, rows, at, start, seq
        self.raw = ArChunks(_ptr(seq), _ptr(start), _ptr(at), n, rows)
        self.ref = ctypes.byref(self.raw)


class Rotary:
    """Rotary positions (ar_rotary): device int32 `positions` [axes][rows], or None (the cache row in every axis);
    `sections`: the frequencies of each axis, adding up to head_size / 2."""

    def __init__(self, theta: float, positions=None, sections=(), layout: int = ROPE_SECTIONS):
        sections = list(sections)
        if len(sections) > 4:
            raise ValueError("at most 4 rotary axes")
        self.positions = positions
        self.raw = ArRotary(theta, _ptr(positions), len(sections), layout, (ctypes.c_int32 * 4)(*sections))
        self.ref = ctypes.byref(self.raw)


class PagedCache:
    """A pool of cache pages and the sequences on them (ar_pages).  Buffers that are not given are allocated, and the
    cache starts empty; given ones are taken as they are and stay the caller's."""

    def __init__(self, ctx: HipContext, layers: int, pages: int, kv_heads: int, head_size: int, seqs: int, max_pages: int,
                 page_rows: int = 64, dtype: int = DTYPE_F32, k=None, v=None, table=None, rows=None, refs=None):
        if dtype not in ELEM_BYTES:
            raise ValueError(f"unknown dtype {dtype}")
        self.ctx, self.dtype = ctx, dtype
        self.layers, self.pages, self.kv_heads, self.head_size = layers, pages, kv_heads, head_size
        self.seqs, self.max_pages, self.page_rows = seqs, max_pages, page_rows
        self._own, self._work, self._need = [], [], {}  # (_work: the last is in use; _need: work bytes by kind of call)

        def take(buf, nbytes, fill):
            if buf is not None or nbytes == 0:
                return buf
            buf = ctx.allocate(nbytes)
            self._own.append(buf)
            if fill is not None:
                buf.upload(np.full(nbytes // 4, fill, np.int32))
            return buf

        pool = layers * pages * kv_heads * page_rows * head_size * ELEM_BYTES[dtype]
        try:
            self.k, self.v = take(k, pool, None), take(v, pool, None)
            self.table = take(table, seqs * max_pages * 4, -1)
            self.rows = take(rows, seqs * 4, 0)
            self.refs = take(refs, pages * 4, 0)
        except Exception:  # (out of memory: nothing of a cache that does not come to be stays)
            for buf in self._own:
                buf.free()
            raise
        self.raw = ArPages(_ptr(self.k), _ptr(self.v), _ptr(self.table), _ptr(self.rows), _ptr(self.refs), dtype,
                           layers, pages, kv_heads, page_rows, head_size, seqs, max_pages)
        self.ref = ctypes.byref(self.raw)

    def close(self):
        """Frees the buffers this cache allocated; calls after it are refused."""
        for buf in self._own + self._work:
            buf.free()
        self._own, self._work = [], []
        self.raw.k = self.raw.v = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _scratch(self, need):
        """The cache's work space, of at least `need` bytes."""
        if not self._work or self._work[-1].nbytes < need:
            self._work.append(self.ctx.allocate(max(need, 2 * self._work[-1].nbytes if self._work else 0)))
        return self._work[-1]

    def _work_bytes(self, key, ask):
        """Work bytes of a kind of call, by `ask(bytes)` where they are not known.  Some are kept, not all that
        there ever were: a server's row counts differ from step to step."""
        need = self._need.get(key)
        if need is None:
            b = ctypes.c_size_t()
            check(ask(ctypes.byref(b)))
            need = b.value
            if len(self._need) >= KEPT_SIZES:
                self._need.clear()
            self._need[key] = need
        return need

    def _table_scratch(self, n):
        return self._scratch(self._work_bytes(n, lambda b: lib().ar_hip_pages_work(self.ref, n, b)))

    def grow(self, chunks: Chunks, missing=None):
        """Room for the chunks' rows at their sequences' ends; fills chunks.at (ar_hip_pages_grow)."""
        w = self._table_scratch(chunks.n)
        check(lib().ar_hip_pages_grow(self.ctx.handle, self.ref, chunks.ref, _ptr(missing), w.ptr, w.nbytes))

    def trim(self, seq, keep, n: int):
        """Sequences keep their first keep[i] rows, None: none (ar_hip_pages_trim)."""
        check(lib().ar_hip_pages_trim(self.ctx.handle, self.ref, _ptr(seq), _ptr(keep), n))

    def fork(self, src, dst, n: int):
        """Sequence dst[i] becomes what src[i] was, on the same pages (ar_hip_pages_fork)."""
        w = self._table_scratch(n)
        check(lib().ar_hip_pages_fork(self.ctx.handle, self.ref, _ptr(src), _ptr(dst), n, w.ptr, w.nbytes))

    def compact(self, live=None):
        """Moves the used pages to the front of the pool (ar_hip_pages_compact)."""
        w = self._table_scratch(0)
        check(lib().ar_hip_pages_compact(self.ctx.handle, self.ref, _ptr(live), w.ptr, w.nbytes))

    def copy(self, to: "PagedCache", src, dst, n: int):
        """Page src[i] of this pool becomes page dst[i] of `to`, in every layer (ar_hip_pages_copy).  A cache of another
        context on the same device: the host waits for that context's queued work before the copy and for the copy
        after it, so that it has its place in both streams; on another device: refused."""
        other = to.ctx is not self.ctx
        if other:
            if to.ctx.index != self.ctx.index:
                raise ValueError(f"pages of device {self.ctx.index} cannot be copied to device {to.ctx.index}")
            to.ctx.synchronize()
        check(lib().ar_hip_pages_copy(self.ctx.handle, self.ref, to.ref, _ptr(src), _ptr(dst), n))
        if other:
            self.ctx.synchronize()

    def write(self, layer: int, chunks: Chunks, q, k, v, q_out, heads: int, rotary: Rotary, act_dtype: int = DTYPE_F32,
              q_stride: int = 0, kv_stride: int = 0, q_norm=None, k_norm=None, eps: float = 1e-6, qk_norm_mode: int = 0):
        """QK-norm, rotary positions, keys and values into the pages, queries to q_out (ar_hip_pages_write).  A stride
        of 0: rows one after another."""
        check(lib().ar_hip_pages_write(self.ctx.handle, self.ref, layer, chunks.ref, _ptr(q), _ptr(k), _ptr(v),
                                       q_stride or heads * self.head_size, kv_stride or self.kv_heads * self.head_size,
                                       heads, _ptr(q_norm), _ptr(k_norm), eps, qk_norm_mode, rotary.ref, _ptr(q_out),
                                       act_dtype))

    def attention(self, layer: int, chunks: Chunks, q, out, heads: int, act_dtype: int = DTYPE_F32):
        """Causal attention of the chunks' rows over their sequences' pages (ar_hip_attention_paged)."""
        w = self._scratch(self._work_bytes(
            (chunks.n, chunks.rows, chunks.start is None, heads),
            lambda b: lib().ar_hip_attention_paged_work(self.ctx.handle, self.ref, chunks.ref, heads, b)))
        check(lib().ar_hip_attention_paged(self.ctx.handle, self.ref, layer, chunks.ref, _ptr(q), act_dtype, heads,
                                           _ptr(out), w.ptr, w.nbytes))
