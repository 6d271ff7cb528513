"""GPU checks of every kernel of the 8-bit path's products (int8_shapes.py; test_int8_shapes.py checks that it has them all),
against sums in whole numbers; tolerances as test_gpu_int8.py derives them."""
import numpy as np
import pytest

import int8_reference as ref
from int8_reference import HALF, U
from int8_shapes import GATED, STORED
from test_gpu_int8 import CODE, EPILOGUE, Eights, Floats, ops  # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu


def _eights(ctx, r, rows, k, std, stride, pad):
    q = r.integers(-127, 128, (rows, k), dtype=np.int8)
    return Eights(ctx, rows, k, stride, q, (std / 73 * np.exp(r.uniform(-1, 1, rows))).astype(np.float32), pad), q


def _scales(e):
    return e.sbuf.download(np.float32, e.rows).astype(np.float64)


def _check(got, want, off, out):
    off = (off + (HALF[out] if out != "f32" else 0) * (np.abs(want) + off)) * (1 + 8 * U)
    bad = ~(np.abs(got.astype(np.float64) - want) <= off)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5])


def _same_in_small_batches(ctx, ops, a, aq, w, w2, bias, c, got, epilogue, out):  # noqa: F811
    """The first and last rows by themselves, which other kernels compute: the same bits."""
    m, k = aq.shape
    for rows in ([0], list(range(max(m - 9, 0), m))):
        part = Eights(ctx, len(rows), k, 0, aq[rows], _scales(a)[rows])
        to = Floats(ctx, c.values[rows], out)
        ops.gemm(part.raw, w.raw, to, epilogue=EPILOGUE[epilogue], W2=w2.raw if w2 else None, bias=bias, c_dtype=CODE[out])
        ctx.synchronize()
        assert (to.get() == got[rows]).all()


@pytest.mark.parametrize("m,n,k", STORED)
def test_stored_and_residual_products(ctx, ops, m, n, k):  # noqa: F811
    r = np.random.default_rng([m, n, k])
    k16 = -(-k // 16) * 16
    a, aq = _eights(ctx, r, m, k, 1.0, k16 + 16, 99)  # (of the bytes behind k one side's may be anything)
    w, wq = _eights(ctx, r, n, k, 1 / np.sqrt(k), k16 + 32, 0)
    p = ref.sums(aq, wq)
    p *= _scales(a)[:, None]
    p *= _scales(w)
    size = np.abs(p)
    bias = Floats(ctx, r.standard_normal((1, n)), "f32")
    before = r.standard_normal((m, n), np.float32)
    for epilogue, out, b, ldc in (("store", "f32", bias, n + 5), ("store", "bf16", None, n + n % 2), ("residual", "f32", None, n),
                                  ("residual", "bf16", None, n + 3)):
        c = Floats(ctx, before, out, ldc, 0)
        ops.gemm(a.raw, w.raw, c, epilogue=EPILOGUE[epilogue], bias=b, c_dtype=CODE[out], ldc=ldc)
        ctx.synchronize()
        got = c.get()
        want = p + (c.values if epilogue == "residual" else b.values.astype(np.float64) if b else 0)
        _check(got, want, 3 * U * size + U * np.abs(want), out)
        if out == "bf16" or b:
            _same_in_small_batches(ctx, ops, a, aq, w, None, b, c, got, epilogue, out)


@pytest.mark.parametrize("m,n,k", GATED)
def test_gated_products(ctx, ops, m, n, k):  # noqa: F811
    r = np.random.default_rng([m, n, k, 2])
    k16 = -(-k // 16) * 16
    a, aq = _eights(ctx, r, m, k, 1.0, k16, 0)
    w, wq = _eights(ctx, r, n, k, 2 / np.sqrt(k), k16 + 16, 44)
    w2, w2q = _eights(ctx, r, n, k, 1 / np.sqrt(k), k16 + 16, -9)
    g = ref.sums(aq, wq) * _scales(a)[:, None] * _scales(w)
    want = ref.silu(g)
    want *= ref.sums(aq, w2q) * _scales(a)[:, None] * _scales(w2)
    off = (6 * np.abs(g) + 32) * U * np.abs(want) + 2.0 ** -120
    for out, ldc in (("f32", n + 3), ("bf16", n + n % 2)):
        c = Floats(ctx, np.zeros((m, n), np.float32), out, ldc, 0)
        ops.gemm(a.raw, w.raw, c, epilogue=EPILOGUE["gated"], W2=w2.raw, c_dtype=CODE[out], ldc=ldc)
        ctx.synchronize()
        got = c.get()
        _check(got, want, off, out)
        _same_in_small_batches(ctx, ops, a, aq, w, w2, None, c, got, "gated", out)
