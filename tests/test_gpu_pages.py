"""GPU checks of the paged cache (common_amd.pages, include/ar_pages.h) against numpy in 64 bits.

Tolerances, per output value, u = 2^-24 (half a step of fp32) and r the half step of a 16-bit result (bf16 2^-8,
fp16 2^-11):
  attention: a score is a sum of head_dim products, off by at most 32 u S with S the largest sum of |q k| / sqrt(hd)
      (sums in chains, whose errors add up as a random walk: sqrt(128) < 32); a weight is off by twice that relative
      to itself and the sums over keys by 32 u again: (64 u S + 32 u) W with W = sum of weight |value|.  bf16
      activations: queries are given in bf16, weights rounded to 16 bits add r W, the output's rounding r |out|.
  write: norm, product and rotation in fp32: angles are exact to a double's rounding and then rounded to fp32 (2 u of
      at most pi each for sin and cos, 4 u with their own error), 16 u of the head's largest value; storing adds r.
Table calls and copies are exact.
"""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_reference as ref
from common_amd import hardware as hw
from common_amd import pages as pg

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
CODE = {"f32": hw.DTYPE_F32, "f16": hw.DTYPE_F16, "bf16": hw.DTYPE_BF16}


def _rng(seed):
    return np.random.default_rng(seed)


def _i32(ctx, values):
    return ctx.to_device(np.asarray(values, np.int32))


class Pool:
    """A cache of random values with random tables, on the device and in numpy."""

    def __init__(self, ctx, rng, dtype, layers, kv, hd, P, lengths, seqs=None, cols=None, spare=3, fill=None):
        self.ctx, self.dtype, self.P = ctx, dtype, P
        seqs = seqs or len(lengths)
        need = [-(-n // P) for n in lengths]
        cols = cols or max(need + [1])
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((seqs, cols), -1, np.int32)
        self.rows = np.zeros(seqs, np.int32)
        for i, n in enumerate(need):
            self.table[i, :n], order = order[:n], order[n:]
            self.rows[i] = lengths[i]
        self.refs = np.zeros(pages, np.int32)
        self.refs[self.table[self.table >= 0]] = 1
        shape = (layers, pages, kv, P, hd)
        self.k, self.v = (ref.to_bits(rng.standard_normal(shape) if fill is None else np.full(shape, fill), dtype)
                          for _ in range(2))
        self.upload(layers, pages, kv, hd, seqs, cols)

    def upload(self, layers, pages, kv, hd, seqs, cols):
        b = {n: self.ctx.to_device(getattr(self, n)) for n in ("k", "v", "table", "rows", "refs")}
        self.buf = b
        self.cache = pg.PagedCache(self.ctx, layers, pages, kv, hd, seqs, cols, page_rows=self.P, dtype=CODE[self.dtype], **b)

    def set(self, name, value):
        setattr(self, name, value)
        self.buf[name].upload(value)

    def down(self, name):
        a = getattr(self, name)
        return self.buf[name].download(a.dtype, a.size).reshape(a.shape)

    def free(self):
        self.cache.close()
        for b in self.buf.values():
            b.free()

    def seen(self, layer, seq):
        """(keys, known), (values, known) of a sequence's whole table row, 64 bits."""
        out = []
        for pool in (self.k, self.v):
            L, kv, hd = self.table.shape[1] * self.P, pool.shape[2], pool.shape[4]
            x, known = np.zeros((L, kv, hd)), np.zeros(L, bool)
            if 0 <= seq < len(self.table):
                for c, page in enumerate(self.table[seq]):
                    if 0 <= page < len(self.refs):
                        x[c * self.P:(c + 1) * self.P] = ref.values(pool[layer, page]).transpose(1, 0, 2)
                        known[c * self.P:(c + 1) * self.P] = True
            out.append((x, known))
        return out


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _attend(ctx, pool, layer, at, counts, q, act, heads, seq=None, extra=2, one_each=False):
    """The call with `extra` rows behind the last chunk; returns [rows, heads, hd] float64 and checks those rows."""
    total, hd = sum(counts), q.shape[2]
    host = ref.to_bits(np.concatenate([q, np.full((extra, heads, hd), np.nan)]), act)
    mark = np.full(host.shape, 0x4321 if act == "bf16" else 7.25, ref.STORED[act])
    qd, od = ctx.to_device(host), ctx.to_device(mark)
    bufs = [qd, od, _i32(ctx, at)] + ([] if one_each else [_i32(ctx, _starts(counts))])
    sq = _i32(ctx, seq) if seq is not None else None
    ch = pg.Chunks(len(counts), total + extra, at=bufs[2], start=None if one_each else bufs[3], seq=sq)
    pool.cache.attention(layer, ch, qd, od, heads, CODE[act])
    ctx.synchronize()
    got = od.download(host.dtype, host.size).reshape(host.shape)
    np.testing.assert_array_equal(got[total:], mark[total:])
    for b in bufs + ([sq] if sq else []):
        b.free()
    return ref.values(got[:total])


def _check_attention(got, pool, layer, at, counts, q, act, heads, seq=None):
    starts = _starts(counts)
    pairs = [pool.seen(layer, i if seq is None else seq[i]) for i in range(len(counts))]
    qv = ref.values(ref.to_bits(q, act))
    want = ref.attention([qv[starts[i]:starts[i + 1]] for i in range(len(counts))], [p[0] for p in pairs],
                         [p[1] for p in pairs], at, counts, heads)
    r = HALF_STEP[act]
    for i, (out, mag, big) in enumerate(want):
        g = got[starts[i]:starts[i + 1]]
        tol = (64 * U * big + 32 * U + r) * mag + r * np.abs(out)
        bad = ~(np.abs(g - out) <= tol)
        assert not bad.any(), (i, np.argwhere(bad)[:4].tolist(), g[bad][:4], out[bad][:4], tol[bad][:4])


TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,P", [(4, 2, 64, 16), (8, 8, 128, 32), (10, 2, 128, 64), (7, 1, 64, 128), (16, 2, 128, 256)])
def test_attention_one_token_each(ctx, act, dtype, heads, kv, hd, P):
    """Decode: one row of each sequence, contexts from none to several pages, ends inside a page and on its border."""
    r = _rng(heads * hd + P)
    at = [0, 1, P - 1, P, 2 * P - 1, 40, 63, 64, 65, 300, 1000]
    pool = Pool(ctx, r, dtype, 2, kv, hd, P, [a + 1 for a in at])
    q = r.standard_normal((len(at), heads, hd))
    got = _attend(ctx, pool, 1, at, [1] * len(at), q, act, heads, one_each=True)
    _check_attention(got, pool, 1, at, [1] * len(at), q, act, heads)
    pool.free()


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,P,at,counts", [
    (4, 2, 64, 16, [0, 5, 100], [1, 17, 33]),
    (6, 2, 128, 32, [0, 31, 32, 200], [64, 0, 31, 3]),
    (3, 3, 64, 64, [0], [130]),
    (8, 1, 128, 16, [7, 250], [20, 5]),
    (16, 8, 128, 64, [513], [129]),
    (5, 1, 64, 256, [0, 700, 0], [0, 70, 260]),
])
def test_attention_chunks(ctx, act, dtype, heads, kv, hd, P, at, counts):
    r = _rng(sum(at) + sum(counts) + hd)
    pool = Pool(ctx, r, dtype, 1, kv, hd, P, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), heads, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, heads)
    _check_attention(got, pool, 0, at, counts, q, act, heads)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("scale", [1e-3, 8.0])
def test_attention_flat_and_peaked_scores(ctx, act, dtype, scale):
    """Scores next to zero (every key counts alike) and scores of tens (one key takes all)."""
    r = _rng(3)
    pool = Pool(ctx, r, dtype, 1, 2, 128, 32, [700, 260])
    q = scale * r.standard_normal((41, 4, 128))
    got = _attend(ctx, pool, 0, [699, 220], [1, 40], q, act, 4)
    _check_attention(got, pool, 0, [699, 220], [1, 40], q, act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_split_long_context(ctx, act, dtype, hd):
    """Few rows over long contexts (the keys are split over blocks), beside an empty and a short one."""
    r = _rng(hd)
    at, counts = [6000, 0, 9, 3333], [1, 1, 2, 5]
    pool = Pool(ctx, r, dtype, 1, 2, hd, 64, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), 4, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    _check_attention(got, pool, 0, at, counts, q, act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [70, 3, 40, 33]])
def test_attention_of_rows_on_no_page(ctx, act, dtype, counts):
    """Entries of -1 and outside the pool hide their rows; a sequence without any, an unknown one and a chunk that is
    not in the cache see nothing and give zeros."""
    r = _rng(11)
    at = [500, 80, 130, -1]
    pool = Pool(ctx, r, dtype, 1, 2, 64, 16, [571, 83, 170, 33])
    t = pool.table.copy()
    t[0, 3:9] = -1
    t[0, 31] = len(pool.refs)
    t[0, 32] = -2 ** 31
    t[0, 33] = 2 ** 31 - 1
    t[1] = -1
    pool.set("table", t)
    q = r.standard_normal((sum(counts), 4, 64))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    _check_attention(got, pool, 0, at, counts, q, act, 4)
    n = counts[0]
    assert not got[n:n + counts[1]].any() and not got[n + counts[1] + counts[2]:].any()
    seq = [2, 9, -1, 0]
    got = _attend(ctx, pool, 0, [100, 5, 5, 400], counts, q, act, 4, seq=seq)
    _check_attention(got, pool, 0, [100, 5, 5, 400], counts, q, act, 4, seq=seq)
    pool.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("hd,at,counts", [(64, [20, 60], [1, 1]), (128, [37, 5], [61, 9]), (64, [600, 90], [140, 3])])
def test_hidden_rows_do_not_reach_the_result(ctx, bad, act, dtype, hd, at, counts):
    """Rows behind the last one, free pages and, for a chunk's earlier rows, its later ones hold NaN or infinities."""
    r = _rng(5)
    pool = Pool(ctx, r, dtype, 1, 2, hd, 16, [a + c + 40 for a, c in zip(at, counts)])
    hidden = ref.to_bits(np.full(1, bad), dtype)[0]
    mid = [a + c // 2 for a, c in zip(at, counts)]  # rows from here on are spoilt; earlier queries must not notice
    for i in range(len(at)):
        for row in range(mid[i] + 1, int((pool.table[i] >= 0).sum()) * 16):
            pool.k[0, pool.table[i, row // 16], :, row % 16] = hidden
            pool.v[0, pool.table[i, row // 16], :, row % 16] = hidden
    for page in np.flatnonzero(pool.refs == 0):
        pool.k[0, page] = pool.v[0, page] = hidden
    pool.set("k", pool.k)
    pool.set("v", pool.v)
    q = r.standard_normal((sum(counts), 4, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    starts = _starts(counts)
    keep = np.concatenate([np.arange(starts[i], starts[i] + mid[i] - at[i] + 1) for i in range(len(at))])
    short = [mid[i] - at[i] + 1 for i in range(len(at))]
    _check_attention(got[keep], pool, 0, at, short, q[keep], act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("hd", [64, 128])
def test_visible_infinity_reaches_only_who_sees_it(ctx, act, dtype, hd):
    """A value of infinity in a chunk's row: later rows' results are infinite in that dim, earlier ones untouched, and
    the other dims of all rows are what they were."""
    r = _rng(17)
    pool = Pool(ctx, r, dtype, 1, 1, hd, 16, [130])
    q = r.standard_normal((90, 2, hd))
    plain = _attend(ctx, pool, 0, [40], [90], q, act, 2)
    v = pool.v.copy()
    v[0, pool.table[0, 100 // 16], 0, 100 % 16, 9] = ref.to_bits(np.full(1, np.inf), dtype)[0]
    pool.set("v", v)
    got = _attend(ctx, pool, 0, [40], [90], q, act, 2)
    assert np.isposinf(got[60:, :, 9]).all()
    got[60:, :, 9] = plain[60:, :, 9]
    np.testing.assert_array_equal(got, plain)
    pool.free()


def test_attention_with_chunk_starts_of_anything_stays_inside(ctx):
    """Starts that descend or leave the rows make empty chunks; the proper ones among them are computed."""
    r = _rng(23)
    pool = Pool(ctx, r, "f16", 1, 2, 64, 16, [60, 60, 60, 60])
    q = r.standard_normal((40, 4, 64))
    for starts in ([0, 10, 5, 20, 40], [0, 10, 90, 95, 99], [-7, 3, 20, 2 ** 31 - 1, 9], [5, 5, 5, 5, 5]):
        qd = ctx.to_device(q.astype(np.float32))
        od = ctx.to_device(np.zeros((40, 4, 64), np.float32))
        at, st = _i32(ctx, [20, 20, 20, 20]), _i32(ctx, starts)
        pool.cache.attention(0, pg.Chunks(4, 40, at=at, start=st), qd, od, 4)
        ctx.synchronize()
        got = od.download(np.float32, q.size)
        assert np.isfinite(got).all()
        for b in (qd, od, at, st):
            b.free()
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads", [2, 64])
@pytest.mark.parametrize("starts,sure", [
    ([0, 10, 25, 90, 95], [0, 1]), ([0, 7, 7, 40, 41], [0, 1, 2]), ([41, 50, 60, 70, 80], []), ([5, 5, 5, 5, 5], []),
    ([3, 20, 20, 33, 40], [0, 2, 3]), ([0, 40, 0, 40, 0], None), ([-7, 3, 20, 2 ** 31 - 1, 9], None)])
def test_attention_leaves_rows_of_no_chunk(ctx, act, dtype, heads, starts, sure):
    """Starts in order whose chunks pass the rows: those chunks are empty, the others are right and nothing else is
    written.  Starts that descend (None): a row is as it was, or finite (zero or an average of values of its pool)."""
    r = _rng(139)
    pool = Pool(ctx, r, dtype, 1, 2, 64, 16, [60, 60, 60, 60])
    q, at = r.standard_normal((40, heads, 64)), [20, 3, 0, 20]
    host = ref.to_bits(q, act)
    mark = np.full(host.shape, 0x4321 if act == "bf16" else 7.25, ref.STORED[act])
    qd, od, a, st = ctx.to_device(host), ctx.to_device(mark), _i32(ctx, at), _i32(ctx, starts)
    pool.cache.attention(0, pg.Chunks(4, 40, at=a, start=st), qd, od, heads, CODE[act])
    ctx.synchronize()
    got = od.download(host.dtype, host.size).reshape(host.shape)
    if sure is None:
        top = np.abs(ref.values(pool.v)).max() * 1.01
        assert ((got == mark) | (np.abs(ref.values(got)) <= top)).all()
    else:
        left = np.ones(40, bool)
        for i in sure:
            x, y = starts[i], starts[i + 1]
            left[x:y] = False
            if y > x:
                _check_attention(ref.values(got[x:y]), pool, 0, at[i:i + 1], [y - x], q[x:y], act, heads, seq=[i])
        np.testing.assert_array_equal(got[left], mark[left])
    for b in (qd, od, a, st):
        b.free()
    pool.free()


def test_attention_repeats_bit_for_bit(ctx):
    r = _rng(29)
    pool = Pool(ctx, r, "f16", 1, 2, 128, 64, [5000, 700])
    q = r.standard_normal((8, 8, 128))
    a = [_attend(ctx, pool, 0, [4999, 690], [1, 7], q, "f32", 8) for _ in range(4)]
    for b in a[1:]:
        np.testing.assert_array_equal(a[0], b)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("counts", [[1, 1, 1], [90, 3, 150]])
def test_unknown_sequences_see_nothing(ctx, act, dtype, counts):
    """Sequence numbers far past the table among proper ones, for one token each and for chunks."""
    r = _rng(41)
    pool = Pool(ctx, r, dtype, 1, 2, 64, 32, [300, 200])
    q = r.standard_normal((sum(counts), 4, 64))
    at = [40, 190, 30]
    for seq in ([2 ** 31 - 1, 1, 0], [2, -2 ** 31, 1], [0, 1 << 29, 1], [2, 3, 4]):
        got = _attend(ctx, pool, 0, at, counts, q, act, 4, seq=seq)
        _check_attention(got, pool, 0, at, counts, q, act, 4, seq=seq)
    pool.free()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("at,counts", [([700, 3], [1, 1]), ([300], [160]), ([5, 90, 0], [70, 1, 40])])
def test_rows_of_very_different_magnitudes(ctx, act, hd, at, counts):
    """fp32 key and value rows from 1e-12 to 1e12, so that the largest value often has next to no weight and the
    largest contribution changes along the keys.  Errors are relative to the contributions' largest dim."""
    r = _rng(43)
    pool = Pool(ctx, r, "f32", 1, 2, hd, 16, [a + c for a, c in zip(at, counts)])
    shape = pool.v.shape[:4] + (1,)
    pool.set("v", (pool.v * 10.0 ** r.uniform(-12, 12, shape)).astype(np.float32))
    pool.set("k", (pool.k * 10.0 ** r.uniform(-12, 0.5, shape)).astype(np.float32))
    q = 3 * r.standard_normal((sum(counts), 4, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    starts = _starts(counts)
    pairs = [pool.seen(0, i) for i in range(len(counts))]
    qv = ref.values(ref.to_bits(q, act))
    want = ref.attention([qv[starts[i]:starts[i + 1]] for i in range(len(counts))], [p[0] for p in pairs],
                         [p[1] for p in pairs], at, counts, 4)
    half = HALF_STEP[act]
    # (bf16 activations over fp32 rows: weights of 11 bits)
    for i, (out, mag, big) in enumerate(want):
        tol = ((64 * U * big + 32 * U + (2.0 ** -11 if act == "bf16" else 0)) * mag).max(-1, keepdims=True) + half * np.abs(out)
        err = np.abs(got[starts[i]:starts[i + 1]] - out)
        assert (err <= tol).all(), (i, (err / tol).max())
    pool.free()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("at,counts", [([700, 3], [1, 1]), ([300], [160]), ([5, 90, 0], [70, 1, 40])])
def test_rows_of_tiny_values(ctx, act, hd, at, counts):
    """fp32 rows near the smallest normal number (keys under queries that bring scores to ordinary size) keep their
    bits."""
    r = _rng(149)
    pool = Pool(ctx, r, "f32", 1, 2, hd, 16, [a + c for a, c in zip(at, counts)])
    pool.set("v", (pool.v * 2.0 ** -116).astype(np.float32))
    pool.set("k", (pool.k * 2.0 ** -118).astype(np.float32))
    q = 2.0 ** 118 * r.standard_normal((sum(counts), 4, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    _check_attention(got, pool, 0, at, counts, q, act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("bf16", "f32"), ("bf16", "bf16"), ("bf16", "f16")])
def test_a_first_tile_of_scores_of_minus_infinity(ctx, act, dtype):
    """Visible keys whose scores are -inf have no weight, also where nothing else has been seen yet.  (bf16 queries: of
    several planes some are 0 or of the other sign, and infinite keys make the row NaN.)"""
    r = _rng(47)
    at, counts = [200, 200], [1, 140]
    pool = Pool(ctx, r, dtype, 1, 1, 64, 64, [201, 340])
    bits = ref.to_bits(np.full(1, -np.inf), dtype)[0]
    for i in range(2):
        pool.k[0, pool.table[i, :2], :, :, 0] = bits
    pool.set("k", pool.k)
    q = r.standard_normal((sum(counts), 4, 64))
    q[..., 0] = 1 + np.abs(q[..., 0])
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    rest = Pool.__new__(Pool)  # the same rows without the first two pages
    rest.__dict__.update(pool.__dict__)
    rest.table = pool.table.copy()
    rest.table[:, :2] = -1
    _check_attention(got, rest, 0, at, counts, q, act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("slope", [0.02, -0.02, 0.15, 1.0, -1.0])
@pytest.mark.parametrize("hd,at,counts", [(64, [900], [1]), (128, [500], [70]), (64, [700, 20, 300], [40, 2, 90])])
def test_scores_that_rise_or_fall_along_the_keys(ctx, act, dtype, slope, hd, at, counts):
    """Rows of one tile whose scores rise, fall or stay: maxima that lag behind and jump, in some rows of a wavefront."""
    r = _rng(97)
    pool = Pool(ctx, r, dtype, 1, 2, hd, 32, [a + c for a, c in zip(at, counts)])
    k = 0.1 * r.standard_normal(pool.k.shape)
    for i in range(len(at)):
        for col, page in enumerate(pool.table[i]):
            if page >= 0:
                k[0, page, :, :, 0] = slope * (col * 32 + np.arange(32)) * np.sqrt(hd)
    pool.set("k", ref.to_bits(k.astype(np.float32), dtype))
    q = 0.5 * r.standard_normal((sum(counts), 8, hd))
    q[..., 0] = r.choice([1.0, 0.0, -1.0, 0.3], q.shape[:2])
    got = _attend(ctx, pool, 0, at, counts, q, act, 8)
    _check_attention(got, pool, 0, at, counts, q, act, 8)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("at,counts", [([60, 63], [3, 1]), ([40], [90]), ([64, 2 ** 31 - 1, 0], [70, 2, 100])])
def test_rows_past_the_table_see_all_of_it(ctx, act, dtype, at, counts):
    r = _rng(101)
    pool = Pool(ctx, r, dtype, 1, 2, 64, 16, [64] * len(at))
    q = r.standard_normal((sum(counts), 4, 64))
    got = _attend(ctx, pool, 0, at, counts, q, act, 4)
    _check_attention(got, pool, 0, at, counts, q, act, 4)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("case", ["ones", "ones-starts", "mixed", "slots-few", "slots-mixed"])
def test_attention_of_many_chunks(ctx, act, dtype, case):
    """More chunks than a wavefront has lanes, and than one call cuts the keys of; empty ones among them."""
    r = _rng(53)
    n = {"ones": 150, "ones-starts": 150, "mixed": 150, "slots-few": 1100, "slots-mixed": 1100}[case]
    counts = [1] * n
    if case in ("ones-starts", "slots-few"):
        counts = r.integers(0, 3, n).tolist()
    if "mixed" in case:
        counts = [int(r.integers(60, 150)) if i % (7 if n < 1000 else 9) == 3 else int(r.integers(0, 4)) for i in range(n)]
        if case == "mixed":
            counts[70] = 700
    KV, G, hd = 2, 4, 64
    seqs = 5
    lengths = [900, 40, 333, 0, 128]
    pool = Pool(ctx, r, dtype, 1, KV, hd, 32, lengths)
    seq = r.integers(0, seqs, n).tolist()
    at = [max(0, int(r.integers(0, max(1, lengths[s] - c + 1)))) for s, c in zip(seq, counts)]
    if case == "ones":
        seq = None
        pool.free()
        lengths = r.integers(0, 300, n).tolist()
        pool = Pool(ctx, r, dtype, 1, KV, hd, 32, lengths)
        at = [x - 1 for x in lengths]
    total = sum(counts)
    q = r.standard_normal((total, KV * G, hd))
    got = _attend(ctx, pool, 0, at, counts, q, act, KV * G, seq=seq, one_each=case == "ones", extra=0 if case == "ones" else 2)
    pick = [i for i in range(n) if i < 3 or i > n - 4 or i % 13 == 3 or i == 70]  # (the 64-bit reference is slow)
    starts = _starts(counts)
    rows = np.concatenate([np.arange(starts[i], starts[i + 1]) for i in pick])
    some = [counts[i] for i in pick]
    _check_attention(got[rows], pool, 0, [at[i] for i in pick], some, q[rows], act, KV * G,
                     seq=[i if seq is None else seq[i] for i in pick])
    assert np.isfinite(got).all()
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("case", ["long-among-short", "more-than-resident"])
def test_attention_of_uneven_batches(ctx, act, dtype, case):
    """Few-row chunks that fill one resident set of blocks: one long context among short ones, and (beside a chunk of
    many rows) more chunks than there are blocks, for which no length of a split has all tasks resident."""
    r = _rng(131)
    if case == "long-among-short":
        KV, G, counts = 8, 1, [1] * (31 if dtype == "f32" else 63)
        at = r.integers(0, 200, len(counts)).tolist()
        at[17] = 20000
    else:
        KV, G, counts = 32, 1, [1] * 40 + [1500]
        at = r.integers(0, 700, len(counts)).tolist()
        at[-1] = 30
    pool = Pool(ctx, r, dtype, 1, KV, 64, 64, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), KV * G, 64))
    got = _attend(ctx, pool, 0, at, counts, q, act, KV * G)
    starts, pick = _starts(counts), [0, 1, 17, len(counts) - 2, len(counts) - 1]
    rows = np.concatenate([np.arange(starts[i], starts[i + 1]) for i in pick])
    _check_attention(got[rows], pool, 0, [at[i] for i in pick], [counts[i] for i in pick], q[rows], act, KV * G, seq=pick)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_single_tokens_in_longer_row_arrays(ctx, act, dtype):
    """Row arrays of a fixed size: the rows behind the last chunk stay as they are and change no result."""
    r = _rng(157)
    pool = Pool(ctx, r, dtype, 1, 2, 64, 64, [3000, 40, 700])
    at, q = [2999, 39, 5], r.standard_normal((3, 8, 64))
    first = _attend(ctx, pool, 0, at, [1, 1, 1], q, act, 8, one_each=True, extra=0)
    _check_attention(first, pool, 0, at, [1, 1, 1], q, act, 8)
    for extra in (1, 61, 5000):
        np.testing.assert_array_equal(_attend(ctx, pool, 0, at, [1, 1, 1], q, act, 8, one_each=True, extra=extra), first)
    pool.free()


def test_merging_blocks_of_two_row_groups_repeat(ctx):
    """Enough tiles that a merging block takes two groups of rows, whose splits are shared (head size 64): the same bits
    every time, and right."""
    r = _rng(107)
    n = 16
    at, counts = [900 + 37 * i for i in range(n)], [64] * n
    pool = Pool(ctx, r, "bf16", 1, 8, 64, 64, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), 32, 64))
    first = _attend(ctx, pool, 0, at, counts, q, "bf16", 32)
    for _ in range(5):
        np.testing.assert_array_equal(_attend(ctx, pool, 0, at, counts, q, "bf16", 32), first)
    for i in (0, 7, 15):
        _check_attention(first[64 * i:64 * i + 64], pool, 0, at[i:i + 1], [64], q[64 * i:64 * i + 64], "bf16", 32, seq=[i])
    pool.free()


@pytest.mark.parametrize("heads,kv,hd", [(96, 96, 64), (40, 40, 128), (300, 3, 64)])
@pytest.mark.parametrize("counts", [[1, 1], [33, 1]])
def test_attention_of_many_heads(ctx, heads, kv, hd, counts):
    r = _rng(59)
    at = [150, 77]
    pool = Pool(ctx, r, "bf16", 1, kv, hd, 16, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), heads, hd))
    got = _attend(ctx, pool, 0, at, counts, q, "bf16", heads)
    _check_attention(got, pool, 0, at, counts, q, "bf16", heads)
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("at,counts", [([3000, 20], [1, 1]), ([600], [150]), ([10, 5, 900], [90, 1, 30])])
def test_attention_in_place(ctx, act, dtype, at, counts):
    """The output over the queries, whether the keys are cut or not."""
    r = _rng(61)
    pool = Pool(ctx, r, dtype, 1, 2, 64, 64, [a + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), 8, 64))
    apart = _attend(ctx, pool, 0, at, counts, q, act, 8)
    host = ref.to_bits(q, act)
    qd, ad, sd = ctx.to_device(host), _i32(ctx, at), _i32(ctx, _starts(counts))
    pool.cache.attention(0, pg.Chunks(len(counts), len(q), at=ad, start=sd), qd, qd, 8, CODE[act])
    ctx.synchronize()
    np.testing.assert_array_equal(ref.values(qd.download(host.dtype, host.size).reshape(host.shape)), apart)
    for b in (qd, ad, sd):
        b.free()
    pool.free()


@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("at,counts", [([3000, 20, -1], [1, 1, 1]), ([600], [150]), ([10, 1500, 900, 0], [90, 1, 30, 0])])
def test_what_the_work_space_held_means_nothing(ctx, act, dtype, at, counts):
    r = _rng(103)
    pool = Pool(ctx, r, dtype, 1, 2, 128, 64, [max(a, 0) + c for a, c in zip(at, counts)])
    q = r.standard_normal((sum(counts), 8, 128))
    host = ref.to_bits(q, act)
    ad, sd, qd = _i32(ctx, at), _i32(ctx, _starts(counts)), ctx.to_device(host)
    ch = pg.Chunks(len(counts), len(q), at=ad, start=sd)
    need = ctypes.c_size_t()
    hw.check(hw.lib().ar_hip_attention_paged_work(ctx.handle, pool.cache.ref, ch.ref, 8, ctypes.byref(need)))
    got = []
    for fill in (0, 0xFFFFFFFF, 0x7F7FFFFF):  # zeros, NaN, the largest float
        w = ctx.to_device(np.full(-(-need.value // 4), fill, np.uint32))
        od = ctx.allocate(host.nbytes)
        hw.check(hw.lib().ar_hip_attention_paged(ctx.handle, pool.cache.ref, 0, ch.ref, qd.ptr, CODE[act], 8, od.ptr, w.ptr,
                                                 need.value))
        ctx.synchronize()
        got.append(ref.values(od.download(host.dtype, host.size).reshape(host.shape)))
        w.free()
        od.free()
    np.testing.assert_array_equal(got[0], got[1])
    np.testing.assert_array_equal(got[0], got[2])
    _check_attention(got[0], pool, 0, at, counts, q, act, 8)
    for b in (ad, sd, qd):
        b.free()
    pool.free()


def test_attention_refuses_on_a_context(ctx):
    """Work space that is missing, too small or not aligned, and more rows than a launch has blocks for."""
    r = _rng(67)
    pool = Pool(ctx, r, "f16", 1, 2, 64, 16, [3000])
    q, o, at = (ctx.allocate(8 * 4 * 64 * 4) for _ in range(3))
    at.upload(np.zeros(8, np.int32))
    ch = pg.Chunks(1, 1, at=at)
    need = ctypes.c_size_t()
    L = hw.lib()
    hw.check(L.ar_hip_attention_paged_work(ctx.handle, pool.cache.ref, ch.ref, 4, ctypes.byref(need)))
    w = ctx.allocate(need.value + 16)

    def call(work, nbytes, chunks=ch, heads=4):
        rc = L.ar_hip_attention_paged(ctx.handle, pool.cache.ref, 0, chunks.ref, q.ptr, 0, heads, o.ptr, work, nbytes)
        return rc, L.ar_hip_last_error().decode()

    for work, nbytes, word in ((None, need.value, "needed"), (w.ptr, need.value - 1, "needed"), (w.ptr + 8, need.value, "aligned")):
        rc, text = call(work, nbytes)
        assert rc == hw.AR_HIP_ERR_INVALID and word in text, text
    assert call(w.ptr, need.value)[0] == 0
    assert call(w.ptr, 0, pg.Chunks(1, 0, at=at, start=at))[0] == 0  # no rows: nothing to do
    many = pg.Chunks(1, 1 << 22, at=at, start=at)
    rc = L.ar_hip_attention_paged_work(ctx.handle, pool.cache.ref, many.ref, 1 << 10, ctypes.byref(need))
    assert rc == hw.AR_HIP_ERR_INVALID and "too many" in L.ar_hip_last_error().decode()
    ctx.synchronize()
    for b in (q, o, at, w):
        b.free()
    pool.free()


def test_two_contexts_at_once(ctx):
    """One pool read on two streams at the same time, each with its own work space."""
    r = _rng(71)
    pool = Pool(ctx, r, "bf16", 1, 2, 128, 64, [4000, 900, 2500])
    at, counts = [3990, 890, 2490], [10, 1, 1]
    q = r.standard_normal((12, 8, 128))
    want = _attend(ctx, pool, 0, at, counts, q, "bf16", 8)
    host = ref.to_bits(q, "bf16")
    with hw.HipContext(0) as other:
        sides = []
        for c in (ctx, other):
            cache = pg.PagedCache(c, 1, len(pool.refs), 2, 128, 3, pool.table.shape[1], page_rows=64, dtype=CODE["bf16"],
                                  **pool.buf)
            sides.append((c, cache, c.to_device(host), c.allocate(host.nbytes), _i32(c, at), _i32(c, _starts(counts))))
        for _ in range(20):
            for c, cache, qd, od, ad, sd in sides:
                cache.attention(0, pg.Chunks(3, 12, at=ad, start=sd), qd, od, 8, CODE["bf16"])
        for c, cache, *bufs in sides:
            c.synchronize()
            np.testing.assert_array_equal(ref.values(bufs[1].download(host.dtype, host.size).reshape(host.shape)), want)
        for c, cache, *bufs in sides:
            cache.close()
            for b in bufs:
                b.free()
    pool.free()


# ---- write -------------------------------------------------------------------------------------------

SECTIONS = {1: (1,), 2: (5, 3), 3: (6, 5, 5), 4: (4, 4, 4, 4)}


def _sections(half, axes):
    s = [half * x // sum(SECTIONS[axes]) for x in SECTIONS[axes]]
    s[0] += half - sum(s)
    if axes == 3:
        s = [half - 2 * (half // 3), half // 3, half // 3]
    return s


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,P,axes,inter,mode,norm,stacked", [
    (4, 2, 64, 16, 1, False, "head", True, True),
    (6, 2, 128, 32, 3, False, "head", True, False),
    (7, 7, 64, 64, 3, True, "whole", True, True),
    (32, 8, 128, 16, 4, True, "head", True, True),
    (40, 40, 64, 256, 2, False, "whole", True, False),
    (5, 1, 128, 32, 2, True, "head", False, True),
])
def test_write(ctx, act, dtype, heads, kv, hd, P, axes, inter, mode, norm, stacked):
    r = _rng(heads + hd + axes)
    at, counts = [0, 15, 200, 31], [20, 1, 40, 0]
    total, extra = sum(counts), 3
    pool = Pool(ctx, r, dtype, 2, kv, hd, P, [a + c for a, c in zip(at, counts)])
    before = pool.k.copy(), pool.v.copy()
    q, k, v = (r.standard_normal((total + extra, n, hd)).astype(np.float32) for n in (heads, kv, kv))
    gq = (1 + 0.1 * r.standard_normal((heads, hd))).astype(np.float32) if norm else None
    gk = (1 + 0.1 * r.standard_normal((kv, hd))).astype(np.float32) if norm else None
    pos = r.integers(0, 5000, (axes, total + extra)).astype(np.int32)
    pos[:, 3] = 2 ** 31 - 1  # a far position
    pos[0, 4] = -12
    sec = _sections(hd // 2, axes)
    bufs = []

    def up(a):
        bufs.append(ctx.to_device(a))
        return bufs[-1]

    if stacked:
        qkv = up(np.concatenate([t.reshape(total + extra, -1) for t in (q, k, v)], 1))
        qs = kvs = (heads + 2 * kv) * hd

        class At:
            def __init__(self, ptr):
                self.ptr = ptr
        qd, kd, vd = (At(qkv.ptr + 4 * hd * x) for x in (0, heads, heads + kv))
    else:
        qd, kd, vd = up(q), up(k), up(v)
        qs = kvs = 0
    mark = np.full((total + extra, heads, hd), 0x4321 if act == "bf16" else 7.25, ref.STORED[act])
    out = up(mark)
    ch = pg.Chunks(4, total + extra, at=up(np.array(at, np.int32)), start=up(_starts(counts)))
    rot = pg.Rotary(1e6, up(pos), sec, pg.ROPE_INTERLEAVED if inter else pg.ROPE_SECTIONS)
    pool.cache.write(1, ch, qd, kd, vd, out, heads, rot, CODE[act], qs, kvs, up(gq) if norm else None,
                     up(gk) if norm else None, 1e-6, 1 if mode == "head" else 0)
    ctx.synchronize()
    got = out.download(mark.dtype, mark.size).reshape(mark.shape)
    np.testing.assert_array_equal(got[total:], mark[total:])
    axis = ref.rotary_axis(hd // 2, axes, sec, inter)
    wq = ref.prepared(q[:total], gq, 1e-6, mode == "head", pos[:, :total], axis, 1e6)
    wk = ref.prepared(k[:total], gk, 1e-6, mode == "head", pos[:, :total], axis, 1e6)

    def close(a, b, t):
        top = np.abs(b).max(-1, keepdims=True)
        assert (np.abs(a - b) <= 16 * U * top + HALF_STEP[t] * (np.abs(b) + 16 * U * top) + 2.0 ** -24).all(), np.abs(a - b).max()

    close(ref.values(got[:total]), wq, act)
    kp, vp = pool.down("k"), pool.down("v")
    starts = _starts(counts)
    for i in range(4):
        for j in range(counts[i]):
            page, off = pool.table[i, (at[i] + j) // P], (at[i] + j) % P
            close(ref.values(kp[1, page, :, off]), wk[starts[i] + j], dtype)
            np.testing.assert_array_equal(vp[1, page, :, off], ref.to_bits(v[starts[i] + j], dtype))
            kp[1, page, :, off], vp[1, page, :, off] = before[0][1, page, :, off], before[1][1, page, :, off]
    np.testing.assert_array_equal(kp, before[0])  # nothing else changed
    np.testing.assert_array_equal(vp, before[1])
    pool.free()
    for b in bufs:
        b.free()


def test_write_drops_rows_on_no_page_and_second_mentions(ctx):
    """Keys and values of rows on no page, past the table, of unknown sequences, of chunks that are not in the cache
    and of a sequence's second chunk are dropped; queries are prepared all the same; positions default to cache rows."""
    r = _rng(31)
    pool = Pool(ctx, r, "f32", 1, 1, 64, 16, [48, 48, 48])
    t = pool.table.copy()
    t[1, 1] = -1
    t[2, 0] = len(pool.refs)
    pool.set("table", t)
    seq, at, counts = [1, 2, 0, 9, 1, 0], [14, 10, 40, 0, 0, -1], [5, 8, 20, 2, 6, 3]
    n = sum(counts)
    k, v, q = (r.standard_normal((n, h, 64)).astype(np.float32) for h in (1, 1, 2))
    bufs = [ctx.to_device(x) for x in (q, k, v, np.zeros_like(q), np.array(at, np.int32), _starts(counts),
                                       np.array(seq, np.int32))]
    ch = pg.Chunks(6, n, at=bufs[4], start=bufs[5], seq=bufs[6])
    pool.cache.write(0, ch, bufs[0], bufs[1], bufs[2], bufs[3], 2, pg.Rotary(1e4, None, [32]))
    ctx.synchronize()
    starts = _starts(counts)
    want_k, want_v = pool.k.copy(), pool.v.copy()
    pos = np.array([a + j if a >= 0 else 0 for a, c in zip(at, counts) for j in range(c)])[None]
    axis = np.zeros(32, int)
    pk, pq = ref.prepared(k, None, 0, True, pos, axis, 1e4), ref.prepared(q, None, 0, True, pos, axis, 1e4)
    written = np.zeros(want_k.shape[:4], bool)
    for i, (s, a, c) in enumerate(zip(seq, at, counts)):
        for j in range(c):
            if s in seq[:i] or not 0 <= s < 3 or a < 0 or a + j >= 48:
                continue
            page = t[s, (a + j) // 16]
            if 0 <= page < len(pool.refs):
                want_k[0, page, :, (a + j) % 16], want_v[0, page, :, (a + j) % 16] = pk[starts[i] + j], v[starts[i] + j]
                written[0, page, :, (a + j) % 16] = True
    assert written.sum() == 2 + 2 + 8  # rows 14, 15 of 1; 16, 17 of 2; 40..47 of 0
    got_k = pool.down("k")
    assert np.abs(got_k - want_k).max() <= 16 * U * np.abs(want_k).max()
    np.testing.assert_array_equal(got_k[~written], pool.k[~written])
    np.testing.assert_array_equal(pool.down("v"), want_v)
    got_q = bufs[3].download(np.float32, q.size).reshape(q.shape)
    assert np.abs(got_q - pq).max() <= 16 * U * np.abs(pq).max()
    pool.free()
    for b in bufs:
        b.free()


def test_write_in_place_and_without_queries(ctx):
    r = _rng(37)
    pool = Pool(ctx, r, "f16", 1, 2, 128, 32, [9, 9])
    q, k, v = (r.standard_normal((18, h, 128)).astype(np.float32) for h in (4, 2, 2))
    g = (1 + 0.1 * r.standard_normal((4, 128))).astype(np.float32)
    qd, kd, vd, o, at, st, gd = (ctx.to_device(x) for x in (q, k, v, np.zeros_like(q), np.zeros(2, np.int32),
                                                            np.array([0, 9, 18], np.int32), g))
    ch, rot = pg.Chunks(2, 18, at=at, start=st), pg.Rotary(1e6, None, [64])
    for mode in (0, 1):
        qd.upload(q)
        pool.cache.write(0, ch, qd, kd, vd, o, 4, rot, q_norm=gd, qk_norm_mode=mode)
        k1, v1 = pool.down("k"), pool.down("v")
        pool.set("k", pool.k)
        pool.set("v", pool.v)
        pool.cache.write(0, ch, None, kd, vd, None, 4, rot)
        np.testing.assert_array_equal(pool.down("k"), k1)
        np.testing.assert_array_equal(pool.down("v"), v1)
        pool.cache.write(0, ch, qd, kd, vd, qd, 4, rot, q_norm=gd, qk_norm_mode=mode)
        ctx.synchronize()
        np.testing.assert_array_equal(qd.download(np.float32, q.size), o.download(np.float32, q.size))
    pool.free()
    for b in (qd, kd, vd, o, at, st, gd):
        b.free()


def test_write_rounds_past_fp16_to_infinity(ctx):
    pool = Pool(ctx, _rng(1), "f16", 1, 1, 64, 16, [1])
    k = np.zeros((1, 1, 64), np.float32)
    k[0, 0, :3] = [65519.0, 65520.0, -70000.0]
    kd, at = ctx.to_device(k), _i32(ctx, [0])
    pool.cache.write(0, pg.Chunks(1, 1, at=at), None, kd, kd, None, 1, pg.Rotary(1e6, None, [32]))
    got = pool.down("v")[0, pool.table[0, 0], 0, 0, :3]
    np.testing.assert_array_equal(got, np.array([65504.0, np.inf, -np.inf], np.float16))
    pool.free()
    kd.free()
    at.free()


# ---- tables and pages ----------------------------------------------------------------------------------

def _same(pool, t, copied=True):
    for name in ("table", "rows", "refs"):
        np.testing.assert_array_equal(pool.down(name), getattr(t, name), err_msg=name)
    if copied:
        k, v = pool.k.copy(), pool.v.copy()
        for s, d in t.copied:
            k[:, d], v[:, d] = pool.k[:, s], pool.v[:, s]
        np.testing.assert_array_equal(pool.down("k"), k)
        np.testing.assert_array_equal(pool.down("v"), v)
        pool.k, pool.v = k, v
    t.copied = []
    pool.table, pool.rows, pool.refs = t.table.copy(), t.rows.copy(), t.refs.copy()


def _grow(ctx, pool, t, counts, seq=None):
    n = len(counts)
    at, st, ms = _i32(ctx, [-5] * n), _i32(ctx, _starts(counts)), _i32(ctx, [-5])
    sq = _i32(ctx, seq) if seq is not None else None
    pool.cache.grow(pg.Chunks(n, sum(counts), at=at, start=st, seq=sq), ms)
    want, missing = t.grow(range(n) if seq is None else seq, counts)
    np.testing.assert_array_equal(at.download(np.int32, n), want)
    assert ms.download(np.int32, 1)[0] == missing
    for b in [at, st, ms] + ([sq] if sq else []):
        b.free()
    return want, missing


def _trim(ctx, pool, t, seq, keep):
    n = len(seq)
    sq, kp = _i32(ctx, seq), _i32(ctx, keep) if keep is not None else None
    pool.cache.trim(sq, kp, n)
    t.trim(seq, keep)
    ctx.synchronize()
    sq.free()
    if kp:
        kp.free()


def _fork(ctx, pool, t, src, dst):
    a, b = _i32(ctx, src), _i32(ctx, dst)
    pool.cache.fork(a, b, len(src))
    t.fork(src, dst)
    ctx.synchronize()
    a.free()
    b.free()


def _tables(pool):
    return ref.Tables(pool.table, pool.rows, pool.refs, pool.P)


@pytest.mark.parametrize("dtype,kv,hd,P", [("f32", 2, 64, 16), ("bf16", 1, 128, 64), ("f16", 8, 128, 256)])
def test_grow_fork_trim_step_by_step(ctx, dtype, kv, hd, P):
    """Sequences share pages, grow apart, and are cut back; tables, counts and copied pages after every call."""
    r = _rng(P)
    pool = Pool(ctx, r, dtype, 2, kv, hd, P, [P + 3, 2 * P, 5, 0], seqs=9, cols=6, spare=14)
    t = _tables(pool)
    _fork(ctx, pool, t, [0, 0, 1, 2, 3], [4, 5, 6, 7, 8])
    _same(pool, t)
    _grow(ctx, pool, t, [1, 2, P, 0, P + 1, 1, 1, 2, 1])        # all sharers of one page in one call: the last keeps it
    _same(pool, t)
    _fork(ctx, pool, t, [4, 5], [5, 4])                          # sources that are targets
    _same(pool, t)
    _grow(ctx, pool, t, [3, 1], [5, 4])
    _same(pool, t)
    _trim(ctx, pool, t, [0, 4, 5, 8, 1], [P + 1, 2, -7, 0, 10 ** 9])
    _same(pool, t)
    _trim(ctx, pool, t, [6, 7, 6], None)
    _same(pool, t)
    assert (t.refs >= 0).all()
    pool.free()


def test_grow_without_enough_pages_or_columns(ctx):
    r = _rng(2)
    pool = Pool(ctx, r, "f32", 1, 1, 64, 16, [20, 20, 7, 30, 0], seqs=8, cols=4, spare=5)
    t = _tables(pool)
    _fork(ctx, pool, t, [0, 0], [5, 6])
    _same(pool, t)
    # 5 free pages; chunk 3 has no columns left, chunk 4 wants more than there is, 5 shares its page with 0 and 6
    at, missing = _grow(ctx, pool, t, [10, 13, 2, 40, 64, 1, 1, 0])
    assert missing > 0 and at[3] == -1 and at[4] == -1
    _same(pool, t)
    at, _ = _grow(ctx, pool, t, [1, 1, 1, 1, 1], [7, 7, -1, 8, 7])
    assert at[0] == 0 and (at[1:] == -1).all()
    _same(pool, t)
    pool.free()


def test_sharers_of_a_page_when_the_pool_runs_out(ctx):
    """Three sequences on one last page and one free page: the first leaves it, the second cannot, so the third may
    not write on it either."""
    pool = Pool(ctx, _rng(4), "f32", 1, 1, 64, 16, [5], seqs=3, cols=2, spare=1)
    t = _tables(pool)
    _fork(ctx, pool, t, [0, 0], [1, 2])
    at, missing = _grow(ctx, pool, t, [1, 1, 1])
    assert at.tolist() == [5, -1, -1] and missing == 1
    _same(pool, t)
    at, missing = _grow(ctx, pool, t, [1, 1], [2, 0])
    assert at.tolist() == [-1, 6] and missing == 1
    _same(pool, t)
    pool.free()


def test_fork_passes_over_unknown_and_repeated_entries(ctx):
    pool = Pool(ctx, _rng(6), "f32", 1, 1, 64, 16, [40, 17, 3], seqs=5, cols=3, spare=2)
    t = _tables(pool)
    _fork(ctx, pool, t, [0, 9, 1, -1, 2, 0, 1], [3, 4, 4, 1, 3, 7, 1])
    _same(pool, t)
    assert t.rows.tolist() == [40, 17, 3, 40, 17]
    pool.free()


@pytest.mark.parametrize("lengths,pages_spare", [([70, 3, 150, 0, 33], 9), ([16], 0), ([5], 1), ([16] * 40, 200)])
def test_compact(ctx, lengths, pages_spare):
    r = _rng(len(lengths))
    pool = Pool(ctx, r, "bf16", 3, 2, 64, 16, lengths, cols=12, spare=pages_spare)
    t = _tables(pool)
    if len(lengths) > 2:
        _fork(ctx, pool, t, [0], [1])
        _same(pool, t)
    live = _i32(ctx, [-1])
    for _ in range(2):  # the second time nothing is left to move
        pool.cache.compact(live)
        ctx.synchronize()
        want = t.compact()
        assert live.download(np.int32, 1)[0] == want == (t.refs > 0).sum()
        assert (t.refs[:want] > 0).all()
        _same(pool, t)
    live.free()
    pool.free()


@pytest.mark.parametrize("seed,P,spare,cols", [(1, 16, 3, 6), (2, 16, 12, 4), (3, 64, 40, 9), (4, 256, 6, 3)])
def test_table_calls_in_any_order(ctx, seed, P, spare, cols):
    """Sequences that come, share, grow, run out of pages, are cut back and moved: every call against the reference,
    and the counts against the table."""
    r = _rng(1000 + seed)
    seqs = 7
    pool = Pool(ctx, r, ["f16", "f32", "bf16", "f32"][seed - 1], 1, 1, 64, P, [P + 5, 2 * P, 3, 0], seqs=seqs, cols=cols, spare=spare)
    t = _tables(pool)
    for step in range(60):
        kind = r.integers(0, 8)
        some = r.permutation(seqs)[:r.integers(1, seqs + 1)].tolist()
        if kind < 4:
            counts = [int(r.choice([0, 1, 1, 2, P - 1, P, P + 1, 2 * P])) for _ in some]
            if kind == 0:  # (one of them twice)
                some, counts = some + some[:1], counts + [1]
            _grow(ctx, pool, t, counts, some)
        elif kind < 6:
            keep = [int(r.choice([0, 1, P - 1, P, P + 1, 3 * P])) for _ in some] if r.integers(0, 3) else None
            _trim(ctx, pool, t, some, keep)
        elif kind == 6:
            _fork(ctx, pool, t, r.integers(-1, seqs + 1, len(some)).tolist(), r.integers(0, seqs, len(some)).tolist())
        else:
            pool.cache.compact(None)
            t.compact()
            ctx.synchronize()
        _same(pool, t)
        held = np.bincount(t.table[t.table >= 0], minlength=len(t.refs))
        np.testing.assert_array_equal(held, t.refs)
    pool.free()


def test_copy_between_pools(ctx):
    r = _rng(8)
    a = Pool(ctx, r, "f16", 3, 2, 128, 32, [320], spare=2)
    b = Pool(ctx, r, "f16", 3, 2, 128, 32, [640], spare=1)
    n, m = len(a.refs), len(b.refs)
    src, dst = [0, 5, 5, n, 3, -1, 7, 2], [4, 9, 1, 2, 4, 8, m, m - 1]
    sd, dd = _i32(ctx, src), _i32(ctx, dst)
    a.cache.copy(b.cache, sd, dd, len(src))
    ctx.synchronize()
    k, v = b.k.copy(), b.v.copy()
    for s, d in ((0, 4), (5, 9), (5, 1), (2, m - 1)):
        k[:, d], v[:, d] = a.k[:, s], a.v[:, s]
    np.testing.assert_array_equal(b.down("k"), k)
    np.testing.assert_array_equal(b.down("v"), v)
    np.testing.assert_array_equal(a.down("k"), a.k)
    for x in (sd, dd):
        x.free()
    a.free()
    b.free()


def test_copy_to_a_cache_of_another_context(ctx):
    """The other context's queued work on the target pages comes before the copy, its later work after it."""
    r = _rng(151)
    with hw.HipContext(0) as other:
        a, b, c = (Pool(x, r, "f32", 4, 8, 128, 64, [64 * 60], spare=4) for x in (ctx, other, other))
        pages = len(a.refs)
        all_pages = [_i32(ctx, r.permutation(pages)) for _ in range(2)]
        assert ctx.index == other.index == 0
        for _ in range(3):
            for k in range(4):  # (each of 67 MB of keys and as much of values)
                c.cache.copy(b.cache, all_pages[0], all_pages[0], pages)
            a.cache.copy(b.cache, all_pages[1], all_pages[1], pages)
            b.cache.copy(c.cache, all_pages[0], all_pages[0], pages)
            other.synchronize()
            for x, y in ((b, a), (c, a)):
                np.testing.assert_array_equal(x.down("k"), a.k)
                np.testing.assert_array_equal(x.down("v"), a.v)
            c.set("k", c.k)
            c.set("v", c.v)
        for x in all_pages:
            x.free()
        for x in (a, b, c):
            x.free()


def test_copy_within_a_pool(ctx):
    pool = Pool(ctx, _rng(9), "f32", 2, 1, 64, 16, [160], spare=2)
    src, dst = [0, 1, 2, 3, 3, 6], [7, 0, 8, 8, 9, 6]  # target 0 is a source, target 8 is named twice, 6 is its own
    sd, dd = _i32(ctx, src), _i32(ctx, dst)
    pool.cache.copy(pool.cache, sd, dd, len(src))
    ctx.synchronize()
    k, v = pool.k.copy(), pool.v.copy()
    for s, d in ((0, 7), (2, 8), (3, 9)):
        k[:, d], v[:, d] = pool.k[:, s], pool.v[:, s]
    np.testing.assert_array_equal(pool.down("k"), k)
    np.testing.assert_array_equal(pool.down("v"), v)
    for x in (sd, dd):
        x.free()
    pool.free()


def test_many_entries(ctx):
    """As many chunks as a call takes, over a pool of more pages than one pass of its search covers."""
    n = 4096
    r = _rng(10)
    lengths = r.integers(0, 20, n).tolist()
    pool = Pool(ctx, r, "f32", 1, 1, 64, 16, lengths, cols=3, spare=2 * n)
    t = _tables(pool)
    _grow(ctx, pool, t, r.integers(0, 25, n).tolist(), r.permutation(n).tolist())
    _same(pool, t)
    _trim(ctx, pool, t, r.permutation(n).tolist(), r.integers(0, 30, n).tolist())
    _same(pool, t)
    pool.free()


# ---- all of them together ------------------------------------------------------------------------------

@pytest.mark.parametrize("act,dtype", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_serving_loop_matches_whole_sequences(ctx, act, dtype):
    """Prompts in chunks, a fork, single tokens and a rolled-back tail, with a compaction between: every row's
    attention equals that over the sequence's own rows kept in plain arrays."""
    r = _rng(77)
    H, KV, hd, P, L, theta = 4, 2, 64, 16, 2, 1e6
    cache = pg.PagedCache(ctx, L, 40, KV, hd, 4, 8, page_rows=P, dtype=CODE[dtype])
    gq, gk = ((1 + 0.1 * r.standard_normal((n, hd))).astype(np.float32) for n in (H, KV))
    gqd, gkd = ctx.to_device(gq), ctx.to_device(gk)
    kept = [[(np.zeros((0, KV, hd)), np.zeros((0, KV, hd))) for _ in range(L)] for _ in range(4)]
    axis = np.zeros(hd // 2, int)
    ms = _i32(ctx, [0])
    half = HALF_STEP[act]

    def step(seqs, counts):
        total = sum(counts)
        at, st, sq = _i32(ctx, [-1] * len(seqs)), _i32(ctx, _starts(counts)), _i32(ctx, seqs)
        ch = pg.Chunks(len(seqs), total, at=at, start=st, seq=sq)
        cache.grow(ch, ms)
        assert ms.download(np.int32, 1)[0] == 0
        first = at.download(np.int32, len(seqs))
        assert first.tolist() == [len(kept[s][0][0]) for s in seqs]
        pos = np.concatenate([np.arange(a, a + c) for a, c in zip(first, counts)])[None]
        for layer in range(L):
            qkv = r.standard_normal((total, H + 2 * KV, hd)).astype(np.float32)
            d = ctx.to_device(qkv)

            class At:
                def __init__(self, ptr):
                    self.ptr = ptr
            q, k, v = (At(d.ptr + 4 * hd * x) for x in (0, H, H + KV))
            qo, o = (ctx.allocate(total * H * hd * 4) for _ in range(2))
            w = (H + 2 * KV) * hd
            cache.write(layer, ch, q, k, v, qo, H, pg.Rotary(theta, None, [hd // 2]), CODE[act], w, w, gqd, gkd, 1e-6, 1)
            cache.attention(layer, ch, qo, o, H, CODE[act])
            ctx.synchronize()
            got = ref.values(o.download(ref.STORED[act], total * H * hd).reshape(total, H, hd))
            # (from the queries as they were handed on, and the keys as the formula has them)
            qv = ref.values(qo.download(ref.STORED[act], total * H * hd).reshape(total, H, hd))
            pk = ref.prepared(qkv[:, H:H + KV], gk, 1e-6, True, pos, axis, theta)
            starts = _starts(counts)
            for i, s in enumerate(seqs):
                a, b = starts[i], starts[i + 1]
                kk = np.concatenate([kept[s][layer][0], ref.values(ref.to_bits(pk[a:b], dtype))])
                vv = np.concatenate([kept[s][layer][1], ref.values(ref.to_bits(qkv[a:b, H + KV:], dtype))])
                kept[s][layer] = (kk, vv)
                known = np.ones(len(kk), bool)
                (out, mag, big), = ref.attention([qv[a:b]], [(kk, known)], [(vv, known)], [first[i]], [b - a], H)
                # a key next to the middle between two stored values may be rounded the other way: a whole step of S
                step_k = 2 * HALF_STEP[dtype] / 8 if dtype != "f32" else 0
                tol = (64 * U * big + 64 * U + half + step_k * big) * mag + half * np.abs(out)
                assert (np.abs(got[a:b] - out) <= tol).all(), (s, layer, np.abs(got[a:b] - out).max())
            for x in (d, qo, o):
                x.free()
        for x in (at, st, sq):
            x.free()

    def fork(s, d):
        a, b = _i32(ctx, [s]), _i32(ctx, [d])
        cache.fork(a, b, 1)
        ctx.synchronize()
        kept[d] = list(kept[s])
        a.free()
        b.free()

    def trim(s, n):
        a, b = _i32(ctx, [s]), _i32(ctx, [n])
        cache.trim(a, b, 1)
        ctx.synchronize()
        kept[s] = [(k[:n], v[:n]) for k, v in kept[s]]
        a.free()
        b.free()

    step([0, 1], [37, 5])
    step([1, 0], [40, 1])
    fork(0, 2)
    step([0, 1, 2], [1, 1, 1])
    step([2, 0], [20, 3])
    trim(1, 0)
    trim(0, 39)
    cache.compact()
    step([0, 1, 2], [1, 30, 1])
    for _ in range(3):
        step([2, 1, 0], [1, 1, 1])
    ctx.synchronize()
    cache.close()
    for x in (gqd, gkd, ms):
        x.free()


def test_offsets_past_32_bits(ctx):
    """The second layer of pools of 5.2 GB: rows written to the last pages, moved by a copy, attended to from one
    token and from a chunk."""
    r = _rng(83)
    KV, hd, P, pages, H = 8, 128, 64, 20000, 16
    lengths, counts = [190, 300], [1, 70]
    cache = pg.PagedCache(ctx, 2, pages, KV, hd, 2, 6, page_rows=P, dtype=CODE["bf16"])
    table = np.full((2, 6), -1, np.int32)
    table[0, :3], table[1, :5] = [19990, 19999, 19985], [19980, 19998, 19970, 19991, 19960]
    td = ctx.to_device(table)
    moved = [19998, 19985]
    rows = sum(lengths)
    k, v = (r.standard_normal((rows, KV, hd)).astype(np.float32) for _ in range(2))
    kd, vd, at, st = ctx.to_device(k), ctx.to_device(v), _i32(ctx, [0, 0]), _i32(ctx, _starts(lengths))
    cache.raw.table = td.ptr
    cache.write(1, pg.Chunks(2, rows, at=at, start=st), None, kd, vd, None, H, pg.Rotary(1e6, None, [hd // 2]))
    pos = np.concatenate([np.arange(n) for n in lengths])[None]
    pk = ref.values(ref.to_bits(ref.prepared(k, None, 0, True, pos, np.zeros(hd // 2, int), 1e6), "bf16"))
    pv = ref.values(ref.to_bits(v, "bf16"))
    q = r.standard_normal((sum(counts), H, hd))
    host = ref.to_bits(q, "bf16")
    qd, od = ctx.to_device(host), ctx.allocate(host.nbytes)
    first = [n - c for n, c in zip(lengths, counts)]
    at2, st2 = _i32(ctx, first), _i32(ctx, _starts(counts))
    src, dst = _i32(ctx, moved), _i32(ctx, [3, 19997])
    outs = []
    for step in range(2):
        if step:
            cache.copy(cache, src, dst, 2)
            t2 = table.copy()
            t2[table == moved[0]], t2[table == moved[1]] = 3, 19997
            ctx.synchronize()
            td.upload(t2)
        for i in (0, 1):  # one token, then the chunk (few rows, then tiles)
            one = pg.Chunks(1, counts[i], at=_At(at2, i), start=_At(st2, 0) if i == 0 else _i32(ctx, [0, counts[1]]),
                            seq=_i32(ctx, [i]))
            row = sum(counts[:i]) * H * hd * 2
            cache.attention(1, one, _At(qd, row // 4), _At(od, row // 4), H, CODE["bf16"])
        ctx.synchronize()
        outs.append(ref.values(od.download(np.uint16, host.size).reshape(host.shape)))
    np.testing.assert_array_equal(outs[0], outs[1])
    qv, ks, cs = ref.values(host), _starts(lengths), _starts(counts)
    for i in range(2):
        known = np.ones(lengths[i], bool)
        kk, vv = pk[ks[i]:ks[i + 1]], pv[ks[i]:ks[i + 1]]
        (out, mag, big), = ref.attention([qv[cs[i]:cs[i + 1]]], [(kk, known)], [(vv, known)], [first[i]], [counts[i]], H)
        half, step_k = HALF_STEP["bf16"], 2 * HALF_STEP["bf16"] / 8  # (keys near the middle of two stored values)
        tol = (64 * U * big + 32 * U + half + step_k * big) * mag + half * np.abs(out)
        assert (np.abs(outs[0][cs[i]:cs[i + 1]] - out) <= tol).all()
    cache.close()


class _At:
    """A buffer's int32 at an index."""

    def __init__(self, buf, index):
        self.ptr = buf.ptr + 4 * index


def test_grow_and_write_with_chunk_starts_of_anything_stay_inside(ctx):
    """Starts that descend or leave the rows make empty chunks; nothing outside the sequences' pages changes."""
    r = _rng(89)
    for starts in ([0, 10, 5, 20, 40], [0, 10, 90, 95, 99], [-7, 3, 20, 2 ** 31 - 1, 9], [0, 40, 0, 40, 0]):
        pool = Pool(ctx, r, "f32", 1, 1, 64, 16, [20, 7, 0, 33], cols=8, spare=20)
        t = _tables(pool)
        counts = [b - a if a >= 0 and b > a and b <= 40 else 0 for a, b in zip(starts, starts[1:])]
        at, st, ms = _i32(ctx, [-5] * 4), _i32(ctx, starts), _i32(ctx, [-5])
        ch = pg.Chunks(4, 40, at=at, start=st)
        pool.cache.grow(ch, ms)
        want, missing = t.grow(range(4), counts)
        np.testing.assert_array_equal(at.download(np.int32, 4), want)
        assert ms.download(np.int32, 1)[0] == missing
        _same(pool, t)
        x = [ctx.to_device(r.standard_normal((40, n, 64)).astype(np.float32)) for n in (2, 1, 1, 2)]
        pool.cache.write(0, ch, x[0], x[1], x[2], x[3], 2, pg.Rotary(1e4, None, [32]))
        ctx.synchronize()
        free = pool.refs == 0
        for name in ("k", "v"):
            np.testing.assert_array_equal(pool.down(name)[:, free], getattr(pool, name)[:, free])
            got = pool.down(name)
            for s, n in enumerate([20, 7, 0, 33]):  # rows that were there before
                for row in range(n):
                    page = pool.table[s, row // 16]
                    np.testing.assert_array_equal(got[0, page, :, row % 16], getattr(pool, name)[0, page, :, row % 16])
        pool.free()
        for b in x + [at, st, ms]:
            b.free()


CHILD = r"""
import ctypes, sys
sys.path.insert(0, ROOT)
import numpy as np
from common_amd import hardware as hw, pages as pg
with hw.HipContext(0) as ctx:
    i32 = lambda v: ctx.to_device(np.asarray(v, np.int32))
    H, KV, hd = 4, 2, 64
    with pg.PagedCache(ctx, 2, 12, KV, hd, 3, 5, page_rows=16) as cache, pg.PagedCache(ctx, 2, 9, KV, hd, 0, 0, page_rows=16) as other:
        at, st, ms = i32([-1, -1]), i32([0, 40, 45]), i32([0])
        ch = pg.Chunks(2, 45, at=at, start=st)
        q, k, v, o = (ctx.to_device(np.ones((45, n, hd), np.float32)) for n in (H, KV, KV, H))
        cache.grow(ch, ms)
        cache.write(0, ch, q, k, v, q, H, pg.Rotary(1e4, i32(np.zeros(90)), [20, 12]))
        cache.attention(0, ch, q, o, H)
        cache.fork(i32([0]), i32([2]), 1)
        cache.trim(i32([1]), i32([2]), 1)
        cache.compact(ms)
        cache.copy(other, i32([0]), i32([1]), 1)
        ctx.synchronize()
        n = ctypes.c_ulonglong()
        hw.check(hw.lib().ar_hip_pointer_checks(ctypes.byref(n)))
        print("checked", n.value)
        short = ctx.allocate(44 * H * hd * 4)
        # (the last int32 of a whole number of 4 KB: HIP gives a few bytes a longer range than was asked for)
        class end: ptr = short.ptr + 44 * H * hd * 4 - 4
        for call in (lambda: cache.attention(0, ch, q, short, H), lambda: cache.attention(0, ch, short, o, H),
                     lambda: cache.write(0, ch, q, short, v, q, H, pg.Rotary(1e4, None, [32]), kv_stride=H * hd),
                     lambda: cache.write(0, ch, q, k, v, q, H, pg.Rotary(1e4, i32(np.zeros(44)), [32])),
                     lambda: cache.trim(end, end, 2)):
            try:
                call()
                print("passed")
            except Exception as e:
                print("refused", "leaves its allocation" in str(e))
        ctx.synchronize()
"""


def test_pointer_checks_cover_the_paged_calls():
    """AR_HIP_CHECK_PTRS=1 (read once per process: a child): every call passes, and is refused when a buffer is short."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", "ROOT = %r\n" % root + CHILD], env=dict(os.environ, AR_HIP_CHECK_PTRS="1"),
                       capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, p.stderr[-3000:]
    lines = p.stdout.split("\n")
    assert lines[0].startswith("checked") and int(lines[0].split()[1]) > 40, p.stdout
    assert lines[1:6] == ["refused True"] * 5, p.stdout


TIMED = """
import torch
import perf.operators as cases

def outputs(o):
    return o if isinstance(o, dict) else {"out": o}

listed = {c["name"]: c for c in cases.listed()}
a = torch.ones(8192, 8192, device="cuda")
for name in ("write-image-prompt", "copy-few", "turnover-6", "attention-chunk-f32"):
    print(name, flush=True)
    case = listed[name]
    want = outputs(cases.run(cases.prepare(case, 5)))
    torch.cuda.synchronize()
    cases.own = True
    cases.run(cases.prepare(case, 6))  # (the context is made)
    torch.cuda.synchronize()
    for _ in range(4):  # some 30 ms, ahead of the inputs
        a @ a
    got = outputs(cases.run(cases.prepare(case, 5)))
    torch.cuda.synchronize()
    cases.own = False
    for key, w in want.items():
        # half a step of 16-bit results on either side; fp32 sums: (64 u S + 32 u) W with S below 20 and W below 1
        w, g = w.double(), got[key].double()
        tol = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}.get(want[key].dtype, 0.0) * w.abs() + 1e-4
        assert want[key].is_floating_point() or (w == g).all(), (name, key)
        assert ((g - w).abs() <= tol).all(), (name, key, float((g - w).abs().max()))
print("ok")
"""


def test_timed_cases_wait_for_their_inputs():
    """The timed cases' inputs are made on torch's stream while the context has its own: the first call on new inputs
    finds them whole, with work still queued on torch's stream when they are made."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", TIMED], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr
