"""GPU checks of the 8-bit path at the ends of fp32's range, against numpy in 64 bits.

Tolerances, u = 2^-24, r the half step of the result's type (bf16 2^-8, fp32 u), relative, for results that are normal numbers:
  product: the sum's conversion and the two products by scales u each, bias and residual u of the result, then r; gated
      (6 |gate| + 32) u of the result in all, then r (test_gpu_int8.py derives both).
"""
import numpy as np
import pytest

import int8_reference as ref
from int8_reference import HALF, U
from test_gpu_int8 import CODE, EPILOGUE, Eights, Floats, Product, _eights_agree, ops  # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu
NORMAL = 2.0 ** -126  # the smallest normal number of fp32 and bf16


def _scales(e, values):
    e.sbuf.upload(np.ascontiguousarray(values, np.float32))


def _far_scales(p, r):
    """Scales of tokens from 2^97 on, of outputs so small that the products are ordinary numbers: scaleA * sum is past fp32 for
    many of them, scaleA * scaleW * sum for none.  Every third token stays ordinary.  Gated: gates of up to some tens."""
    gated = p.epilogue == "gated"
    sa = np.ldexp(r.uniform(1, 1.99, p.m), r.integers(97, 112 if gated else 128, p.m))
    sa[1::3] = r.uniform(0.5, 2, len(sa[1::3]))
    if p.m > 4:
        sa[3] = -sa[3]
    _scales(p.a, sa)
    _scales(p.w, np.ldexp(r.uniform(1, 2, p.n), r.integers(-126, -124 if gated else -100, p.n)))
    if gated:
        _scales(p.w2, np.ldexp(r.uniform(1, 2, p.n), r.integers(-126, -100, p.n)))


FAR = [(1, 2560, 4096), (3, 40, 64), (16, 100, 300), (20, 5000, 200), (64, 512, 1024), (100, 260, 500), (300, 700, 640),
       (700, 5000, 300), (64, 2560, 9728)]


@pytest.mark.parametrize("m,n,k", FAR)
@pytest.mark.parametrize("epilogue,out", [("store", "f32"), ("residual", "bf16"), ("gated", "f32"), ("gated", "bf16")])
def test_token_scales_near_fp32s_largest(ctx, ops, m, n, k, epilogue, out):  # noqa: F811
    """scaleA * sum may be past fp32 where scaleA * scaleW * sum is not."""
    r = np.random.default_rng([m, n, k])
    p = Product(ctx, m, n, k, epilogue, out, bias=epilogue == "store")
    _far_scales(p, r)
    p.run(ops)
    ctx.synchronize()
    sa = p.scales(p.a)[:, None]
    g = ref.sums(p.aq, p.wq) * sa * p.scales(p.w)
    near = np.abs(g) <= 80  # (of the gated ones)
    if epilogue == "gated":
        want = np.where(near, ref.sums(p.aq, p.w2q) * sa * p.scales(p.w2) * ref.silu(np.where(near, g, 0)), 0)
        off = (6 * np.abs(g) + 32) * U * np.abs(want)
    else:
        more = p.c.values.astype(np.float64) if epilogue == "residual" else p.bias.values.astype(np.float64)
        want = g + more
        off = 3 * U * np.abs(g) + U * np.abs(want)
    off = off + (HALF[out] if out != "f32" else 0) * (np.abs(want) + off) + NORMAL
    got = p.c.get().astype(np.float64)
    look = near if epilogue == "gated" else np.ones_like(near)
    assert look.mean() > 0.5 and np.abs(want).max() < 2.0 ** 100
    assert (np.abs(got - want) <= off * (1 + 8 * U))[look].all()


@pytest.mark.parametrize("epilogue,out", [("store", "f32"), ("residual", "bf16"), ("gated", "f32"), ("gated", "bf16")])
def test_rows_beside_such_tokens_have_the_same_bits(ctx, ops, epilogue, out):  # noqa: F811
    p = Product(ctx, 150, 300, 700, epilogue, out, bias=epilogue == "store", seed=3)
    plain = p.scales(p.a)
    sa = plain.copy()
    sa[::5] = 2.0 ** 127
    _scales(p.a, np.concatenate([sa, [5.0]]))
    p.run(ops)
    ctx.synchronize()
    got = p.c.get()
    keep = np.arange(150) % 5 != 0
    for rows in (np.nonzero(keep)[0][:7], np.nonzero(keep)[0][:60], np.nonzero(keep)[0]):
        c = Floats(ctx, p.c.values[rows], out)
        a = Eights(ctx, len(rows), 700, 0, p.aq[rows], plain[rows])
        ops.gemm(a.raw, p.w.raw, c, epilogue=EPILOGUE[epilogue], W2=p.w2.raw if p.w2 else None, bias=p.bias,
                 c_dtype=CODE[out])
        ctx.synchronize()
        assert (c.get() == got[rows]).all()
    far = got[~keep]
    alone = Floats(ctx, p.c.values[~keep], out)
    a = Eights(ctx, 30, 700, 0, p.aq[~keep], sa[~keep])
    ops.gemm(a.raw, p.w.raw, alone, epilogue=EPILOGUE[epilogue], W2=p.w2.raw if p.w2 else None, bias=p.bias, c_dtype=CODE[out])
    ctx.synchronize()
    assert np.array_equal(alone.get(), far, equal_nan=True)


@pytest.mark.parametrize("m", [1, 12, 40, 130, 300])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_gates_far_below_zero_before_large_up_projections(ctx, ops, m, out):  # noqa: F811
    """silu(-100) is 100 * 2^-144: no normal number of fp32, but the product with an up projection of 1e30 is."""
    r = np.random.default_rng(m)
    n, k = 200, 128
    p = Product(ctx, m, n, k, "gated", out)
    sa = np.exp(r.uniform(-1, 1, m))
    _scales(p.a, sa)
    sums, sums2 = ref.sums(p.aq, p.wq), ref.sums(p.aq, p.w2q)
    _scales(p.w, np.exp(r.uniform(np.log(20), np.log(400), n)) / np.abs(sums).mean())  # gates to some -1,000
    _scales(p.w2, np.ldexp(r.uniform(1, 2, n), r.integers(0, 100, n)))
    p.run(ops)
    ctx.synchronize()
    g = sums * p.scales(p.a)[:, None] * p.scales(p.w)
    up = sums2 * p.scales(p.a)[:, None] * p.scales(p.w2)
    want = up * ref.silu(g)
    off = (6 * np.abs(g) + 32) * U * np.abs(want)
    off = off + (HALF[out] if out != "f32" else 0) * (np.abs(want) + off) + NORMAL
    far = (g < -87) & (np.abs(want) > 2.0 ** -100)
    assert far.sum() > 5
    got = p.c.get().astype(np.float64)
    past = np.abs(want) > 2.0 ** 128  # (what is past both types' largest is infinite)
    assert (got[past] == np.sign(want[past]) * np.inf).all()
    bad = ~past & ~(np.abs(got - want) <= off * (1 + 8 * U))
    assert not bad.any(), (int(bad.sum()), g[bad][:5], up[bad][:5], got[bad][:5], want[bad][:5])


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_gates_of_minus_infinity_shut_the_up_projection_off(ctx, ops, m, out):  # noqa: F811
    n, k = 96, 256
    one = np.ones((m, k), np.int8)
    a = Eights(ctx, m, k, 0, one, np.ones(m, np.float32))
    w = Eights(ctx, n, k, 0, -np.ones((n, k), np.int8), np.full(n, 3e38, np.float32))
    w2 = Eights(ctx, n, k, 0, np.ones((n, k), np.int8), np.full(n, 1e35, np.float32))
    c = Floats(ctx, np.ones((m, n)), out)
    ops.gemm(a.raw, w.raw, c, epilogue=EPILOGUE["gated"], W2=w2.raw, c_dtype=CODE[out])
    ctx.synchronize()
    assert (c.get() == 0).all()


@pytest.mark.parametrize("n", [40, 2560, 40000])
@pytest.mark.parametrize("yd", ["f32", "bf16", "i8"])
def test_norms_of_rows_near_fp32s_largest(ctx, ops, n, yd):  # noqa: F811
    """Root mean squares past 2^126, whose reciprocals are no normal numbers; within 5 u as all others (test_gpu_int8.py)."""
    r = np.random.default_rng(n)
    a = (r.uniform(2.6e38, 3.4e38, (33, n)) * r.choice([-1, 1], (33, n))).astype(np.float32)
    a[::4, : n // 2] = 0
    a[5] *= np.float32(2.0 ** -3)
    a[6, 1:] = 1
    h, w = Floats(ctx, a, "f32"), Floats(ctx, 1 + 0.3 * r.standard_normal((1, n)), "f32")
    _, want = ref.norm(h.values, None, w.values[0], np.float32(1e-6))
    if yd == "i8":
        out = Eights(ctx, 33, n)
        ops.add_rmsnorm_i8(h, w, 1e-6, out.raw)
        ctx.synchronize()
        _eights_agree(out, want, 5 * U)
    else:
        out = Floats(ctx, np.zeros((33, n)), yd)
        ops.add_rmsnorm(h, w, 1e-6, 33, n, out, y_dtype=CODE[yd])
        ctx.synchronize()
        off = (5 * U + (HALF[yd] if yd != "f32" else 0)) * np.abs(want) * (1 + U) + NORMAL
        assert (np.abs(out.get() - want) <= off).all()
