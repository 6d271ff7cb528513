"""GPU checks of the 8-bit path (common_amd.int8, include/ar_i8.h) against numpy in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32), r the half step of the result's type (bf16 2^-8, fp32 u), all relative:
  quantize: the scale is one division, u.  A number is x times 127 / m, both rounded: within 1/2 + 127 * 2 u of the
      unrounded one in 64 bits.
  norm: the sum h + x is off by u; the root's reciprocal by u and by what the squares of those sums make (u); the two
      products by u each: 5 u, and r where it is stored.  In 8 bits: the scale 6 u, a number 1/2 + 127 * (2 * 5 u + 2 u)
      (the row's largest and the value are both off by 5 u).
  embed: one product, u, then r.
  product: the sum is exact, its conversion and two products by scales are off by u each; bias and residual add u of the
      result; then r.  Gated, with g = p(W), up = p(W2): g and up are off by 3 u, exp(-g) by 3 |g| u from g, |g| u from
      its argument's product, a few u of its own: (6 |g| + 32) u of the result in all, then r.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

import int8_reference as ref
from common_amd import hardware as hw
from common_amd import int8
from int8_reference import HALF, U

pytestmark = pytest.mark.gpu
CODE = {"f32": hw.DTYPE_F32, "bf16": hw.DTYPE_BF16}
NP = {"f32": np.float32, "bf16": np.uint16}
EPILOGUE = {"store": hw.GEMM_STORE, "residual": hw.GEMM_RESIDUAL, "gated": hw.GEMM_SWIGLU}


@pytest.fixture(scope="module")
def ops(ctx):
    o = int8.Int8Ops(ctx)
    yield o
    ctx.synchronize()
    o.close()


def _rng(*seed):
    return np.random.default_rng(list(seed))


class Floats:
    """Float rows on the device, `stride` values apart, `offset` values into their buffer, 3.0 between them."""

    def __init__(self, ctx, a, dtype, stride=0, offset=0):
        rows, n = a.shape
        self.shape, self.dtype, self.stride, self.offset = (rows, n), dtype, stride or n, offset
        host = np.full(offset + rows * self.stride + 7, 3.0, np.float32)
        host[offset:offset + rows * self.stride].reshape(rows, self.stride)[:, :n] = a
        host = ref.to_bits(host, dtype)
        self.buf = ctx.to_device(host)
        self.ptr = self.buf.ptr + offset * host.itemsize
        self.size = host.size
        self.values = self.get()

    def get(self):
        """The values; what lies between and around the rows has to be as it was."""
        host = ref.to_f32(self.buf.download(NP[self.dtype], self.size))
        rows, n = self.shape
        mid = host[self.offset:self.offset + rows * self.stride].reshape(rows, self.stride)
        assert (host[:self.offset] == 3).all() and (host[self.offset + rows * self.stride:] == 3).all()
        assert (mid[:, n:] == 3).all()
        return mid[:, :n].copy()


class Eights:
    """Rows in 8 bits on the device, with bytes of 77 around them (and between n rounded up to 16 and the stride)."""

    def __init__(self, ctx, rows, n, stride=0, q=None, scale=None, pad=0):
        self.rows, self.n, self.n16 = rows, n, -(-n // 16) * 16
        self.stride = stride or self.n16
        host = np.full((rows + 1, self.stride), 77, np.int8)
        if q is not None:
            host[:rows, :n] = q
            host[:rows, n:self.n16] = pad
        self.buf = ctx.to_device(host)
        self.sbuf = ctx.to_device(np.concatenate([np.zeros(rows, np.float32) if scale is None else scale,
                                                  [5.0]]).astype(np.float32))
        self.raw = int8.Int8Rows(ctx, rows, n, q=self.buf, scale=self.sbuf, stride=self.stride)

    def get(self):
        host = self.buf.download(np.int8, (self.rows + 1) * self.stride).reshape(self.rows + 1, self.stride)
        scale = self.sbuf.download(np.float32, self.rows + 1)
        assert (host[self.rows] == 77).all() and (host[:, self.n16:] == 77).all() and scale[-1] == 5
        assert (host[:self.rows, self.n:self.n16] == 0).all()
        return host[:self.rows, :self.n].astype(np.int64), scale[:-1]


def _eights_agree(out, y, off):
    """Rows in 8 bits against rows y in 64 bits that the kernel knew to within `off`, relative."""
    q, scale = out.get()
    want, steps = ref.quantize(y)
    assert np.abs(scale - steps).max(initial=0) <= ((off + U) * steps).max(initial=0)
    assert (np.abs(scale - steps) <= (off + U) * steps).all()
    assert (np.abs(q - want) <= 0.5 + 127 * (2 * off + 2 * U)).all()


# ---- rows ---------------------------------------------------------------------------------------------

SIZES = [(1, 1, 0, 0), (3, 7, 0, 0), (5, 64, 0, 0), (2, 2560, 0, 0), (7, 2561, 0, 0), (9, 4096, 4104, 0), (4, 768, 769, 3),
         (2, 9728, 9736, 8), (33, 100, 112, 0), (3, 16384, 0, 0), (2, 32769, 0, 0), (1, 131071, 0, 0), (1030, 40, 0, 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,stride,offset", SIZES)
def test_quantize(ctx, ops, rows, n, stride, offset, dtype):
    r = _rng(rows, n, 1)
    a = r.standard_normal((rows, n)) * np.exp(r.uniform(-8, 8, (rows, 1)))
    x = Floats(ctx, a, dtype, stride, offset)
    out = Eights(ctx, rows, n, stride=(-(-n // 16) * 16 + 32) if stride else 0)
    ops.quantize(x, out.raw, CODE[dtype], stride)
    ctx.synchronize()
    _eights_agree(out, x.values, 0.0)


@pytest.mark.parametrize("n", [40, 4096, 40000])
def test_quantize_rows_of_zeros_tiny_and_infinite_values(ctx, ops, n):
    a = np.ones((8, n), np.float32)
    a[0] = 0
    a[1] = 2.0 ** -101          # below the smallest that is held
    a[2] = 0
    a[2, n - 1] = -2.0 ** -100  # the smallest
    a[3, n // 2] = np.inf
    a[4, 0] = np.nan
    a[5] = np.float32(3.4028235e38)
    a[6] = -2.0 ** -140         # not normal
    a[7, 3] = -np.inf
    x, out = Floats(ctx, a, "f32"), Eights(ctx, 8, n)
    ops.quantize(x, out.raw)
    y = Floats(ctx, np.zeros((8, n)), "f32")
    ops.embed(out.raw, None, 8, y)
    ctx.synchronize()
    q, s = out.get()
    assert (s[[0, 1, 6]] == 0).all() and (q[[0, 1, 6]] == 0).all()
    assert q[2, n - 1] == -127 and (q[2, :n - 1] == 0).all() and abs(s[2] * 127 / 2.0 ** -100 - 1) <= 2 * U
    assert np.isnan(s[[3, 4, 7]]).all() and (q[[3, 4, 7]] == 0).all()
    assert (q[5] == 127).all() and abs(float(s[5]) * 127 / 3.4028235e38 - 1) <= 2 * U
    got = y.get()
    assert np.isnan(got[[3, 4, 7]]).all() and (got[[0, 1, 6]] == 0).all()


NORMS = [("f32", "f32", "i8"), ("f32", "bf16", "i8"), ("bf16", "bf16", "i8"), ("bf16", "f32", "i8"),
         ("f32", "f32", "f32"), ("f32", "bf16", "bf16"), ("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"),
         ("f32", None, "i8"), ("bf16", None, "i8"), ("bf16", None, "f32"), ("f32", None, "bf16")]


@pytest.mark.parametrize("hd,xd,yd", NORMS)
@pytest.mark.parametrize("rows,n,stride,offset", SIZES)
def test_norm(ctx, ops, rows, n, stride, offset, hd, xd, yd):
    r = _rng(rows, n, 2)
    h = Floats(ctx, r.standard_normal((rows, n)) * np.exp(r.uniform(-3, 3, (rows, 1))), hd, stride, offset)
    x = Floats(ctx, r.standard_normal((rows, n)), xd, stride, offset) if xd else None
    w = Floats(ctx, (1 + 0.3 * r.standard_normal((1, n))), "f32")
    v, y = ref.norm(h.values, x.values if x else None, w.values[0], np.float32(1e-6))
    kind = dict(h_dtype=CODE[hd], x_dtype=CODE[xd or "f32"], h_stride=stride, x_stride=stride)
    if yd == "i8":
        out = Eights(ctx, rows, n)
        ops.add_rmsnorm_i8(h, w, 1e-6, out.raw, x=x, **kind)
        ctx.synchronize()
        _eights_agree(out, y, 5 * U)
    else:
        out = Floats(ctx, np.zeros((rows, n)), yd, stride, offset)
        ops.add_rmsnorm(h, w, 1e-6, rows, n, out, x=x, y_dtype=CODE[yd], y_stride=stride, **kind)
        ctx.synchronize()
        assert (np.abs(out.get() - y) <= (5 * U + (HALF[yd] if yd != "f32" else 0)) * np.abs(y) * (1 + U)).all()
    if x is None:
        assert (h.get() == h.values).all()  # nothing was added
    else:
        assert (np.abs(h.get() - v) <= (U + (HALF[hd] if hd != "f32" else 0)) * np.abs(v) * (1 + HALF[hd])).all()
        assert (x.get() == x.values).all()


@pytest.mark.parametrize("n", [37, 2560, 40000])
def test_norm_over_its_input_and_of_extremes(ctx, ops, n):
    """y may be x; squares past fp32's range; rows of zeros, infinities and NaN."""
    r = _rng(n, 3)
    hv = r.standard_normal((6, n)).astype(np.float32)
    hv[1] *= np.float32(1e30)   # squares beyond fp32
    hv[2] *= np.float32(1e-30)  # ... and below it
    hv[3] = 0
    hv[4, 5] = np.nan
    hv[5, 7] = np.inf
    xv = np.zeros((6, n), np.float32)
    w = Floats(ctx, np.ones((1, n)), "f32")
    for yd in ("f32", "i8"):
        h, x = Floats(ctx, hv, "f32"), Floats(ctx, xv, "f32")
        out = Eights(ctx, 6, n)
        if yd == "f32":
            ops.add_rmsnorm(h, w, 1e-30, 6, n, x, x=x)
        else:
            ops.add_rmsnorm_i8(h, w, 1e-30, out.raw, x=x)
        ctx.synchronize()
        _, want = ref.norm(hv[:4], None, np.ones(n), np.float64(np.float32(1e-30)))
        if yd == "f32":
            got = x.get()
            assert (np.abs(got[:4] - want) <= 5 * U * np.abs(want) * (1 + U)).all()
            assert np.isnan(got[4]).all() and np.isnan(got[5, 7]) and (np.delete(got[5], 7) == 0).all()
        else:
            q, s = out.get()
            q0, s0 = ref.quantize(want)
            assert (np.abs(q[:4] - q0) <= 0.5 + 127 * 12 * U).all() and (np.abs(s[:4] - s0) <= 6 * U * s0).all()
            assert np.isnan(s[4:]).all() and (q[4:] == 0).all()


@pytest.mark.parametrize("yd", ["f32", "bf16"])
@pytest.mark.parametrize("table,n,count,stride,ys", [(5, 1, 3, 0, 0), (100, 768, 8, 0, 0), (37, 2560, 300, 0, 0),
                                                     (64, 100, 65, 160, 103), (9, 5000, 4, 5040, 5001), (3, 40, 2000, 0, 0),
                                                     (50, 264, 4099, 0, 0), (4200, 72, 4200, 0, 0), (7, 33, 4097, 0, 40),
                                                     (6, 9000, 9, 0, 0)])
def test_embed(ctx, ops, table, n, count, stride, ys, yd):
    r = _rng(table, n, 4)
    q, scale = r.integers(-127, 128, (table, n)), np.exp(r.uniform(-9, 3, table)).astype(np.float32)
    t = Eights(ctx, table, n, stride, q, scale)
    tokens = r.integers(0, table, count).astype(np.int32)
    if count > 4:  # outside the table
        tokens[1], tokens[2], tokens[3] = -1, table, 2 ** 31 - 1
    y = Floats(ctx, np.zeros((count, n)), yd, ys)
    ops.embed(t.raw, ctx.to_device(tokens), count, y, CODE[yd], ys)
    some = min(count, table)
    z = Floats(ctx, np.zeros((some, n)), yd, ys)
    ops.embed(t.raw, None, some, z, CODE[yd], ys)
    ctx.synchronize()
    every = q * scale.astype(np.float64)[:, None]
    known = (tokens >= 0) & (tokens < table)
    want = np.where(known[:, None], every[np.where(known, tokens, 0)], 0)
    for got, exact in ((y.get(), want), (z.get(), every[:some])):
        assert (np.abs(got - exact) <= (U + (HALF[yd] if yd != "f32" else 0)) * np.abs(exact) * (1 + U)).all()


def test_more_rows_than_a_launch_takes(ctx, ops):
    """Rows go out in launches of 2^20, for a launch's threads to stay below 2^32."""
    rows = 2 ** 20 + 5
    test_quantize(ctx, ops, rows, 16, 0, 0, "bf16")
    test_norm(ctx, ops, rows, 8, 0, 0, "f32", "bf16", "i8")
    test_norm(ctx, ops, rows, 8, 0, 0, "bf16", "bf16", "f32")
    test_embed(ctx, ops, 7, 8, rows, 0, 0, "f32")
    test_embed(ctx, ops, rows, 8, rows, 0, 0, "bf16")


# ---- products -----------------------------------------------------------------------------------------

class Product:
    """Random rows, the product on the device, and what it has to be."""

    def __init__(self, ctx, m, n, k, epilogue="store", out="f32", bias=False, seed=0, strides=False, pad="w", full=False,
                 gate=2.0):
        r = _rng(m, n, k, seed)
        self.ctx, self.m, self.n, self.k, self.epilogue, self.out = ctx, m, n, k, epilogue, out
        k16 = -(-k // 16) * 16
        lo = -128 if full else -127

        def eights(rows, std, pad_value):
            q = r.integers(lo, 128, (rows, k)).astype(np.int8)
            if full:
                q[:] = -128
            return Eights(ctx, rows, k, k16 + 16 * int(strides) * (1 + rows % 3), q,
                          (std / 73 * np.exp(r.uniform(-1, 1, rows))).astype(np.float32), pad_value), q

        # of the bytes behind k one side's may be anything
        self.a, self.aq = eights(m, 1.0, 99 if pad == "w" else 0)
        self.w, self.wq = eights(n, gate / np.sqrt(k), 0 if pad == "w" else -55)
        self.w2, self.w2q = eights(n, 1.0 / np.sqrt(k), 0 if pad == "w" else 31) if epilogue == "gated" else (None, None)
        if self.w2:
            assert self.w2.stride == self.w.stride
        self.bias = Floats(ctx, r.standard_normal((1, n)), "f32") if bias else None
        self.c = Floats(ctx, r.standard_normal((m, n)), out, n + 5 if strides else 0, 1 if strides else 0)

    def run(self, ops):
        ops.gemm(self.a.raw, self.w.raw, self.c, epilogue=EPILOGUE[self.epilogue], W2=self.w2.raw if self.w2 else None,
                 bias=self.bias, c_dtype=CODE[self.out], ldc=self.c.stride)
        return self

    def scales(self, e):
        return e.sbuf.download(np.float32, e.rows).astype(np.float64)

    def check(self):
        sa = self.scales(self.a)[:, None]
        g = ref.sums(self.aq, self.wq) * sa * self.scales(self.w)
        if self.epilogue == "gated":
            want = ref.sums(self.aq, self.w2q) * sa * self.scales(self.w2) * ref.silu(g)
            off = (6 * np.abs(g) + 32) * U * np.abs(want) + 2.0 ** -120
        else:
            want = g + (self.c.values.astype(np.float64) if self.epilogue == "residual" else
                        self.bias.values.astype(np.float64) if self.bias else 0)
            off = 3 * U * np.abs(g) + U * np.abs(want)
        off = off + (HALF[self.out] if self.out != "f32" else 0) * (np.abs(want) + off)
        got = self.c.get().astype(np.float64)
        bad = ~(np.abs(got - want) <= off * (1 + 8 * U))
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5])
        return got


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 2560, 4096), (2, 17, 100), (5, 130, 33), (8, 300, 2560), (15, 31, 1000), (16, 2048, 768),
          (17, 100, 2049), (32, 257, 640), (33, 640, 129), (48, 96, 9728), (63, 65, 127), (64, 512, 512), (65, 300, 4100),
          (100, 1000, 260), (127, 129, 128), (128, 128, 1024), (129, 127, 1040), (200, 70, 16), (255, 511, 384),
          (256, 256, 2560), (257, 513, 300), (509, 640, 1024), (1000, 257, 192), (1025, 1030, 144), (3, 5000, 48)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("epilogue,out,bias,strides", [("store", "f32", True, False), ("residual", "f32", False, True),
                                                       ("gated", "bf16", False, False), ("store", "bf16", False, True),
                                                       ("residual", "bf16", False, False), ("gated", "f32", False, True)])
def test_product(ctx, ops, m, n, k, epilogue, out, bias, strides):
    p = Product(ctx, m, n, k, epilogue, out, bias, strides=strides, pad="w" if (m + n) % 2 else "a").run(ops)
    ctx.synchronize()
    p.check()


# larger tiles, cut at the last token, output and step, in one round of the CUs and in several (int8_shapes.py has every kind)
LARGE = [(700, 5000, 300), (1025, 8200, 200), (2000, 6100, 150), (1500, 3000, 260), (515, 2600, 1100), (70, 1000, 9000),
         (140, 2500, 5000), (3000, 4100, 140), (4000, 4700, 160), (3900, 4500, 145), (900, 6000, 140), (2750, 9700, 200)]


@pytest.mark.parametrize("m,n,k", LARGE)
@pytest.mark.parametrize("epilogue,out,bias,strides", [("store", "f32", True, False), ("residual", "f32", False, True),
                                                       ("gated", "bf16", False, True), ("store", "bf16", False, True),
                                                       ("residual", "bf16", False, False), ("gated", "f32", False, False)])
def test_large_product(ctx, ops, m, n, k, epilogue, out, bias, strides):
    p = Product(ctx, m, n, k, epilogue, out, bias, strides=strides).run(ops)
    ctx.synchronize()
    p.check()


@pytest.mark.parametrize("m,n", [(1, 40), (20, 33), (130, 140)])
def test_product_of_the_longest_rows_of_the_largest_numbers(ctx, ops, m, n):
    """131,071 products of -128 by -128 are 16,384 short of 2^31."""
    p = Product(ctx, m, n, 131071, full=True).run(ops)
    ctx.synchronize()
    p.check()


@pytest.mark.parametrize("epilogue,out", [("store", "f32"), ("residual", "bf16"), ("gated", "f32"), ("gated", "bf16")])
@pytest.mark.parametrize("n,k", [(520, 1100), (1027, 4096), (96, 9000)])
def test_rows_have_the_same_bits_in_any_batch(ctx, ops, n, k, epilogue, out):
    p = Product(ctx, 700, n, k, epilogue, out, bias=epilogue == "store", seed=5).run(ops)
    ctx.synchronize()
    whole = p.c.get()
    for m0, m in ((0, 1), (3, 2), (0, 9), (100, 16), (11, 30), (40, 64), (64, 128), (0, 300), (600, 100)):
        c = Floats(ctx, p.c.values[m0:m0 + m], out)
        a = Eights(ctx, m, k, 0, p.aq[m0:m0 + m], p.scales(p.a)[m0:m0 + m])
        ops.gemm(a.raw, p.w.raw, c, epilogue=EPILOGUE[epilogue], W2=p.w2.raw if p.w2 else None, bias=p.bias,
                 c_dtype=CODE[out])
        ctx.synchronize()
        assert (c.get() == whole[m0:m0 + m]).all(), m


def test_product_of_no_rows_and_scales_that_are_no_numbers(ctx, ops):
    c = Floats(ctx, np.ones((4, 40)), "f32")
    w = Eights(ctx, 40, 64, 0, np.ones((40, 64), np.int8), np.ones(40, np.float32))
    a = Eights(ctx, 4, 64, 0, np.ones((4, 64), np.int8), np.array([1, np.nan, 0, 2], np.float32))
    ops.gemm(a.raw.first(0), w.raw, c)
    ops.gemm(a.raw, w.raw.first(0), c, ldc=40)
    ctx.synchronize()
    assert (c.get() == 1).all()
    ops.gemm(a.raw, w.raw, c)
    ctx.synchronize()
    got = c.get()
    assert (got[0] == 64).all() and np.isnan(got[1]).all() and (got[2] == 0).all() and (got[3] == 128).all()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_gates_far_from_zero(ctx, ops, m):
    """Gates to +-1000: the sigmoid's ends neither overflow nor lose the sign."""
    p = Product(ctx, m, 300, 256, "gated", "f32", gate=2000.0).run(ops)
    ctx.synchronize()
    p.check()


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_gates_without_end_and_gates_that_are_no_numbers(ctx, ops, m, out):
    """Products beyond fp32: an infinite gate passes the up projection on or shuts it off; NaN stays NaN."""
    n, k = 96, 256
    one = lambda r: np.ones((r, k), np.int8)  # noqa: E731
    gate = one(n)
    gate[1::3] = -1
    scale = np.full(n, 3e38, np.float32)
    scale[2::3] = np.nan
    a = Eights(ctx, m, k, 0, one(m), np.ones(m, np.float32))
    w = Eights(ctx, n, k, 0, gate, scale)
    w2 = Eights(ctx, n, k, 0, one(n), np.full(n, 2.0 ** -8, np.float32))
    c = Floats(ctx, np.ones((m, n)), out)
    ops.gemm(a.raw, w.raw, c, epilogue=hw.GEMM_SWIGLU, W2=w2.raw, c_dtype=CODE[out])
    ctx.synchronize()
    got = c.get()
    assert (got[:, 0::3] == np.inf).all() and (np.abs(got[:, 1::3]) < 2.0 ** -115).all() and np.isnan(got[:, 2::3]).all()


def test_work_space_that_is_missing_short_or_not_aligned_is_refused(ctx, ops):
    import ctypes
    L, b = hw.lib(), ctypes.c_size_t()
    p = Product(ctx, 64, 2560, 9728)
    hw.check(L.ar_hip_gemm_i8_work(ctx.handle, 64, 2560, 9728, hw.GEMM_STORE, ctypes.byref(b)))
    assert b.value > 0
    hw.check(L.ar_hip_gemm_i8_work(ctx.handle, 1, 2560, 9728, hw.GEMM_STORE, ctypes.byref(b)))
    assert b.value == 0
    hw.check(L.ar_hip_gemm_i8_work(ctx.handle, 64, 2560, 9728, hw.GEMM_STORE, ctypes.byref(b)))
    work = ctx.allocate(b.value + 16)
    for ptr, size in ((None, b.value), (work.ptr, b.value - 1), (work.ptr + 8, b.value)):
        rc = L.ar_hip_gemm_i8(ctx.handle, p.a.raw.ref, p.w.raw.ref, None, None, p.c.ptr, hw.DTYPE_F32, 2560, hw.GEMM_STORE,
                              ptr, size)
        assert rc == hw.AR_HIP_ERR_INVALID and b"work space" in L.ar_hip_last_error()
    # any contents will do, and what lies behind the space stays
    host = np.full((b.value + 16) // 4, -7, np.int32)
    work.upload(host)
    hw.check(L.ar_hip_gemm_i8(ctx.handle, p.a.raw.ref, p.w.raw.ref, None, None, p.c.ptr, hw.DTYPE_F32, 2560, hw.GEMM_STORE,
                              work.ptr, b.value))
    ctx.synchronize()
    p.check()
    assert (work.download(np.int32, 4, b.value) == -7).all()


CHECKED = """
import numpy as np
from common_amd import hardware as hw
from common_amd import int8
with hw.HipContext(0) as ctx:
    ops = int8.Int8Ops(ctx)
    x, out = ctx.to_device(np.ones((4, 64), np.float32)), ops.rows(4, 64)
    y = ctx.allocate(4 * 64 * 4)
    ops.quantize(x, out)
    ops.embed(out, None, 4, y)
    ops.gemm(out, out, ctx.allocate(64))
    n = __import__("ctypes").c_ulonglong()
    hw.check(hw.lib().ar_hip_pointer_checks(__import__("ctypes").byref(n)))
    assert n.value >= 9, n.value
    short = ctx.allocate(4 * 64 * 4 - 4)
    for call in (lambda: ops.quantize(short, out), lambda: ops.embed(out, None, 4, short),
                 lambda: ops.add_rmsnorm_i8(short, x, 1e-6, out), lambda: ops.add_rmsnorm_i8(y, x, 1e-6, out, x=short),
                 lambda: ops.add_rmsnorm(y, x, 1e-6, 4, 64, short),
                 lambda: ops.gemm(out, int8.Int8Rows(ctx, 4, 64, q=short, scale=x, stride=256), y),
                 lambda: ops.gemm(out, out, ctx.allocate(60))):
        try:
            call()
        except hw.HardwareException as e:
            assert e.code == hw.AR_HIP_ERR_INVALID and "leaves its allocation" in str(e), e
        else:
            raise AssertionError("not refused")
    ctx.synchronize()
print("refused")
"""


def test_pointer_checks_of_every_call():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CHECKED], cwd=root, env=dict(os.environ, AR_HIP_CHECK_PTRS="1"),
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout + r.stderr


def test_two_contexts_at_once(ctx, ops):
    """Calls of two contexts, queued side by side, on the same rows: nothing between them but the rows."""
    p = Product(ctx, 64, 2560, 9728)
    ctx.synchronize()
    with hw.HipContext(0) as other:
        mine = int8.Int8Ops(other)
        outs = []
        for i in range(6):
            c = Floats(ctx, np.zeros((64, 2560)), "f32")
            outs.append(c)
            (ops if i % 2 else mine).gemm(p.a.raw, p.w.raw, c)
        other.synchronize()
        ctx.synchronize()
        mine.close()
    p.run(ops)
    ctx.synchronize()
    p.check()
    for c in outs:
        assert (c.get() == p.c.get()).all()


# ---- a run of them together ---------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 7, 150])
@pytest.mark.parametrize("res", ["f32", "bf16"])
def test_feed_forward_block_of_a_step(ctx, ops, tokens, res):
    """Embedding, residual norm, gated product, its rows in 8 bits, down product, logits: each call's result against 64
    bits on what the calls before it left, and the whole against the unquantized block."""
    r = _rng(tokens, 7)
    dim, F, V = 200, 330, 500

    def weights(rows, n, std):
        x = Floats(ctx, r.standard_normal((rows, n)) * std, "bf16")
        e = Eights(ctx, rows, n)
        ops.quantize(x, e.raw, hw.DTYPE_BF16)
        return x, e

    (tx, table), (gx, gate), (ux, up), (dx, down) = (weights(V, dim, 1.0), weights(F, dim, 0.1), weights(F, dim, 0.1),
                                                     weights(dim, F, 0.1))
    ids = r.integers(0, V, tokens).astype(np.int32)
    h = Floats(ctx, np.zeros((tokens, dim)), res)
    attn = Floats(ctx, r.standard_normal((tokens, dim)) * 0.3, "f32")
    w = Floats(ctx, 1 + 0.1 * r.standard_normal((1, dim)), "f32")
    x8, act8 = Eights(ctx, tokens, dim), Eights(ctx, tokens, F)
    act = Floats(ctx, np.zeros((tokens, F)), "bf16")
    logits = Floats(ctx, np.zeros((tokens, V)), "f32")
    ops.embed(table.raw, ctx.to_device(ids), tokens, h, CODE[res])
    ctx.synchronize()
    h0 = h.get()
    ops.add_rmsnorm_i8(h, w, 1e-6, x8.raw, x=attn, h_dtype=CODE[res])
    ctx.synchronize()
    h1 = h.get()
    ops.gemm(x8.raw, gate.raw, act, epilogue=hw.GEMM_SWIGLU, W2=up.raw, c_dtype=hw.DTYPE_BF16)
    ops.quantize(act, act8.raw, hw.DTYPE_BF16)
    ops.gemm(act8.raw, down.raw, h, epilogue=hw.GEMM_RESIDUAL, c_dtype=CODE[res])
    ctx.synchronize()
    h2 = h.get()
    ops.add_rmsnorm_i8(h, w, 1e-6, x8.raw, h_dtype=CODE[res])
    ops.gemm(x8.raw, table.raw, logits)
    ctx.synchronize()

    def values(e):
        q, s = e.get()
        return q * s.astype(np.float64)[:, None]

    assert (np.abs(h0 - values(table)[ids]) <= (U + (HALF[res] if res != "f32" else 0)) * np.abs(h0) * 1.01).all()
    v, y = ref.norm(h0, attn.values, w.values[0], np.float32(1e-6))
    assert (np.abs(h1 - v) <= (U + (HALF[res] if res != "f32" else 0)) * np.abs(v) * 1.01).all()
    d = values(act8) @ values(down).T
    want = h1 + d
    assert (np.abs(h2 - want) <= 3 * U * np.abs(d) + (U + (HALF[res] if res != "f32" else 0)) * np.abs(want) * 1.01).all()
    _eights_agree(x8, ref.norm(h2, None, w.values[0], np.float32(1e-6))[1], 5 * U)
    z = values(x8) @ values(table).T
    assert (np.abs(logits.get() - z) <= 4 * U * np.abs(z)).all()
    # the whole against the block without 8 bits: half a step of a row's largest value is 1/254 of it; rows of some
    # hundred values have largest ones of about 3.5 times their root mean square: errors of 3.5 / 254 / sqrt(3) = 0.8 % of
    # each factor, four of them in the gate's and down's products (inputs, weights, twice), the gate's counted twice by
    # its slope: within 6 x 0.8 % of the block's output, which is a part of h
    u = ref.silu(y @ gx.values.astype(np.float64).T) * (y @ ux.values.astype(np.float64).T)
    full = u @ dx.values.astype(np.float64).T
    assert np.linalg.norm(d - full) <= 0.05 * np.linalg.norm(full)
