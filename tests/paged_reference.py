"""The paged cache's calls one step after another in numpy, in 64 bits where they compute (include/ar_pages.h is what
they follow): the tests' reference."""
import numpy as np


def to_bits(a, dtype):
    """fp32 values as the stored type, rounded to nearest even: float32, float16, or bfloat16 as uint16 bits."""
    a = np.asarray(a, np.float32)
    if dtype == "f32":
        return a
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def values(a):
    """Stored values as float64."""
    if a.dtype == np.uint16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


STORED = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


class Tables:
    """table, rows and refs, and the copies that a call makes as (source, target) in `copied`."""

    def __init__(self, table, rows, refs, page_rows):
        self.table, self.rows, self.refs, self.P = table.copy(), rows.copy(), refs.copy(), page_rows
        self.copied = []

    def grow(self, seqs, counts):
        at, named, stuck, wanted = [], set(), False, 0
        free = [i for i in range(len(self.refs)) if self.refs[i] == 0]
        total = len(free)
        waiting = {}  # page -> chunks that have not left it for want of pages
        for s, c in zip(seqs, counts):
            ok = 0 <= s < len(self.rows) and s not in named
            named.add(s)
            ok = ok and self.rows[s] + c <= self.table.shape[1] * self.P
            if not ok:
                at.append(-1)
                continue
            old = int(self.rows[s])
            tail, part = divmod(old, self.P)
            last = int(self.table[s, tail]) if part and c else -1
            shared = last >= 0 and self.refs[last] - waiting.get(last, 0) > 1
            need = -(-(old + c) // self.P) - -(-old // self.P) + shared if c else 0
            wanted += need
            if need and (stuck or need > len(free)):
                stuck = True
                if shared:  # (counted as if it had left, for the sum of what is wanted)
                    waiting[last] = waiting.get(last, 0) + 1
                at.append(-1)
                continue
            if last >= 0 and not need and waiting.get(last):
                at.append(-1)
                continue
            cols = list(range(tail + (1 if part and not shared else 0), -(-(old + c) // self.P))) if c else []
            for k, col in enumerate(cols):
                page = free.pop(0)
                self.table[s, col], self.refs[page] = page, 1
                if shared and k == 0:
                    self.copied.append((last, page))
                    self.refs[last] -= 1
            self.rows[s] = old + c
            at.append(old)
        return np.array(at, np.int32), max(0, wanted - total)

    def trim(self, seqs, keep):
        named = set()
        for i, s in enumerate(seqs):
            if not 0 <= s < len(self.rows) or s in named:
                continue
            named.add(s)
            k = 0 if keep is None else max(int(keep[i]), 0)
            if k >= self.rows[s]:
                continue
            for c in range(-(-k // self.P), -(-int(self.rows[s]) // self.P)):
                if self.table[s, c] >= 0:
                    self.refs[self.table[s, c]] -= 1
                self.table[s, c] = -1
            self.rows[s] = k

    def fork(self, src, dst):
        before, rows, named = self.table.copy(), self.rows.copy(), set()
        n = len(self.rows)
        for s, d in zip(src, dst):
            if not (0 <= s < n and 0 <= d < n) or d in named:
                continue
            named.add(d)
            for page in before[s][before[s] >= 0]:
                self.refs[page] += 1
            for page in before[d][before[d] >= 0]:
                self.refs[page] -= 1
            self.table[d], self.rows[d] = before[s], rows[s]

    def compact(self):
        used = self.refs > 0
        live = int(used.sum())
        movers = [i for i in range(live, len(used)) if used[i]]
        holes = [i for i in range(live) if not used[i]]
        to = np.arange(len(used))
        for m, h in zip(movers, holes):
            to[m] = h
            self.refs[h], self.refs[m] = self.refs[m], 0
            self.copied.append((m, h))
        self.table = np.where(self.table >= 0, to[self.table], -1).astype(np.int32)
        return live


def rotary_axis(half, axes, sections, interleaved):
    if not interleaved:
        return np.repeat(np.arange(axes), sections[:axes])
    return np.array([f % axes if f // axes < sections[f % axes] else 0 for f in range(half)])


def prepared(x, gain, eps, per_head, pos, axis, theta):
    """x [rows, heads, hd] normalised and turned; pos [axes, rows]."""
    x = x.astype(np.float64)
    hd = x.shape[2]
    if gain is not None:
        over = (2,) if per_head else (1, 2)
        x = gain.astype(np.float64).reshape(1, -1, hd) * x / np.sqrt((x * x).mean(over, keepdims=True) + eps)
    f = np.arange(hd // 2)
    a = pos[axis].T.astype(np.float64) * theta ** (-2.0 * f / hd)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    lo, hi = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)


def attention(q, keys, vals, at, counts, heads):
    """q: list of [count, heads, hd]; keys / vals: list of ([rows, kv, hd], known [rows]).  Returns per chunk the
    outputs, the sums of |weight x value| and the largest sum of |q k| / sqrt(hd) over a row's keys."""
    res = []
    for i, n in enumerate(counts):
        k, known = keys[i]
        v, _ = vals[i]
        hd, kv = k.shape[2], k.shape[1]
        out, mag, big = (np.zeros((n, heads, hd)) for _ in range(3))
        for j in range(n):
            see = np.flatnonzero(known[:max(0, at[i] + j + 1)]) if at[i] >= 0 else np.zeros(0, int)
            if not len(see):
                continue
            for h in range(heads):
                kk, vv = k[see, h // (heads // kv)], v[see, h // (heads // kv)]
                s = kk @ q[i][j, h] / np.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[j, h], mag[j, h] = w @ vv, w @ np.abs(vv)
                big[j, h] = (np.abs(kk) @ np.abs(q[i][j, h])).max() / np.sqrt(hd)
        res.append((out, mag, big))
    return res
