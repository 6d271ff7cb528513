"""GPU checks of rows in 8 bits byte by byte: the scale is m / 127 and a byte x * (127 / m), each operation rounded once in
fp32, and the byte to the nearest, halves to even.  Exact: no tolerance."""
import numpy as np
import pytest

import int8_reference as ref
from test_gpu_int8 import CODE, Eights, Floats, ops  # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu


def _bytes(x):
    """(bytes, scales) of fp32 rows in fp32 arithmetic."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(1, keepdims=True)
    return np.rint(x * (np.float32(127) / top)).astype(np.int64), (top / np.float32(127))[:, 0]


def _run(ctx, ops, a, dtype):  # noqa: F811
    x, out = Floats(ctx, a, dtype), Eights(ctx, *a.shape)
    ops.quantize(x, out.raw, CODE[dtype])
    ctx.synchronize()
    return x.values, *out.get()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [254, 300, 2560, 9728, 32768, 40000])
def test_halves_go_to_the_even_number(ctx, ops, n, dtype):  # noqa: F811
    """Rows whose largest magnitude is 127 keep their numbers (the scale and 127 / m are 1): every half between -127 and 127, and
    what lies next to one, which bf16 rounds to it."""
    halves = np.arange(-126.5, 127)
    a = np.stack([np.resize(halves, n), np.resize(np.nextafter(halves, np.inf, dtype=np.float32), n),
                  np.resize(np.nextafter(halves, -np.inf, dtype=np.float32), n)]).astype(np.float32)
    a[:, n // 2] = 127
    a[1, n // 2] = -127
    values, q, scale = _run(ctx, ops, a, dtype)
    want = np.rint(values.astype(np.float64)).astype(np.int64)
    for other in (np.floor(values + 0.5), np.ceil(values - 0.5), np.trunc(values + np.copysign(0.5, values))):
        assert (other[0] != want[0]).sum() > 60  # (what rounds halves in another manner would be seen)
    assert (q == want).all() and (scale == 1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 4096), (257, 768), (65, 2561), (9, 16384), (4, 33000), (2000, 100)])
def test_bytes_and_scales_are_those_of_fp32_arithmetic(ctx, ops, rows, n, dtype):  # noqa: F811
    r = np.random.default_rng([rows, n])
    a = r.standard_normal((rows, n)) * np.exp(r.uniform(-60, 60, (rows, 1)))
    values, q, scale = _run(ctx, ops, a.astype(np.float32), dtype)
    want, steps = _bytes(values)
    assert (q == want).all() and (scale == steps).all()
    assert (np.abs(want - ref.quantize(values)[0]) <= 0.5 + 1e-4).all()  # (the arithmetic is itself that of the definition)


def test_repeated_calls_give_the_same_bytes(ctx, ops):  # noqa: F811
    a = np.random.default_rng(3).standard_normal((700, 2560)).astype(np.float32)
    first = _run(ctx, ops, a, "bf16")
    for _ in range(3):
        again = _run(ctx, ops, a, "bf16")
        assert (again[1] == first[1]).all() and (again[2] == first[2]).all()
