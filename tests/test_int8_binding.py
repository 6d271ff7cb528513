"""CPU checks of what common_amd.int8 does before and after the C calls."""
import pytest

from common_amd import hardware as hw
from common_amd import int8


class _Buf:
    def __init__(self, ptr):
        self.ptr, self.freed = ptr, False

    def free(self):
        self.freed, self.ptr = True, None


class _Context:
    """A context of device `index` that never reaches one: calls that get past the binding are refused by the library."""

    handle = None

    def __init__(self, index=0):
        self.index, self.bufs = index, []

    def allocate(self, nbytes):
        self.bufs.append(_Buf(4096 * (len(self.bufs) + 1)))
        return self.bufs[-1]


def test_rows_taken_from_others_end_with_them():
    """After `close` the memory is gone: rows that share it must not keep its address."""
    ctx = _Context()
    whole = int8.Int8Rows(ctx, 8, 40)
    part = whole.first(5)
    less = part.first(2)
    assert part.raw.q == less.raw.q == whole.raw.q and (part.raw.rows, less.raw.rows) == (5, 2)
    part.close()  # (its own are none: the others stay)
    assert part.raw.q is None and less.raw.q is None and whole.raw.q == 4096 and not any(b.freed for b in ctx.bufs)
    again, kept = whole.first(8), whole.first(3)
    whole.close()
    assert all(b.freed for b in ctx.bufs)
    for rows in (whole, again, kept):
        assert rows.raw.q is None and rows.raw.scale is None
        with int8.Int8Ops(ctx) as ops, pytest.raises(hw.HardwareException, match="null pointer"):
            ops.quantize(_Buf(4096), rows)


def test_rows_outlive_the_ones_they_were_taken_from():
    ctx = _Context()
    part = int8.Int8Rows(ctx, 8, 40).first(5)
    assert part.raw.q == 4096 and not any(b.freed for b in ctx.bufs)


def test_no_rows_are_taken_from_closed_ones():
    """`first` of closed rows allocated new, unset memory for what it took."""
    ctx = _Context()
    whole = int8.Int8Rows(ctx, 8, 40)
    whole.close()
    with pytest.raises(ValueError, match="closed"):
        whole.first(3)
    assert len(ctx.bufs) == 2


CALLS = {
    "quantize": lambda ops, rows, other: ops.quantize(_Buf(4096), other),
    "add_rmsnorm_i8": lambda ops, rows, other: ops.add_rmsnorm_i8(_Buf(4096), _Buf(4096), 1e-6, other),
    "embed": lambda ops, rows, other: ops.embed(other, None, 2, _Buf(4096)),
    "gemm A": lambda ops, rows, other: ops.gemm(other, rows, _Buf(4096)),
    "gemm W": lambda ops, rows, other: ops.gemm(rows, other, _Buf(4096)),
    "gemm W2": lambda ops, rows, other: ops.gemm(rows, rows, _Buf(4096), epilogue=hw.GEMM_SWIGLU, W2=other),
}


@pytest.mark.parametrize("call", sorted(CALLS))
def test_rows_of_another_device_are_refused(call):
    """Their memory is another GPU's; rows of another context on the same device are the caller's to order."""
    ops = int8.Int8Ops(_Context(0))
    rows = int8.Int8Rows(ops.ctx, 8, 40)
    with pytest.raises(ValueError, match="rows of device 1 .* device 0"):
        CALLS[call](ops, rows, int8.Int8Rows(_Context(1), 8, 40))
    assert len(ops.ctx.bufs) == 2  # (no work space was taken for it)
    with pytest.raises(hw.HardwareException, match="ctx is null"):
        CALLS[call](ops, rows, int8.Int8Rows(_Context(0), 8, 40))


@pytest.mark.parametrize("call", sorted(CALLS))
def test_rows_on_given_buffers_need_no_context(call):
    """Rows made without one, on the caller's buffers, are used as before."""
    ops = int8.Int8Ops(_Context(0))
    rows, other = (int8.Int8Rows(None, 8, 40, q=_Buf(4096), scale=_Buf(8192)) for _ in range(2))
    with pytest.raises(hw.HardwareException, match="ctx is null"):
        CALLS[call](ops, rows, other)
