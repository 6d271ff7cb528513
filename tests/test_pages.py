"""CPU checks of the paged cache: its index arithmetic on well-formed arrays and on arrays full of anything (under the
address and undefined-behaviour sanitizers), and the refusals of its calls, which come before anything else."""
import ctypes
import os
import shutil
import subprocess

import pytest

from common_amd import hardware as hw
from common_amd import pages as pg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 4096  # an aligned address that is never read


def test_index_arithmetic_under_sanitizers(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "page_index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-o",
                    exe, os.path.join(ROOT, "tests", "sanitize", "page_index_main.cpp")], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:verify_asan_link_order=0")
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def test_tasks_of_attention_under_sanitizers(tmp_path):
    """How attention cuts its keys: every split of every tile has a task of its own below the number of tasks, and the
    fewest units of a split are found in some 25 questions at any accepted size."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "page_tasks")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-o",
                    exe, os.path.join(ROOT, "tests", "sanitize", "page_tasks_main.cpp")], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:verify_asan_link_order=0")
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def _pages(**over):
    f = dict(k=A, v=2 * A, table=A, rows=A, refs=A, dtype=hw.DTYPE_F32, layers=2, pages=8, kv_heads=2, page_rows=16,
             head_dim=64, seqs=3, max_pages=4)
    f.update(over)
    return pg.ArPages(**f)


def _chunks(**over):
    f = dict(seq=None, start=A, at=A, n=2, rows=5)
    f.update(over)
    return pg.ArChunks(**f)


def _rotary(**over):
    f = dict(theta=1e6, positions=A, axes=3, layout=pg.ROPE_SECTIONS, section=(16, 8, 8, 0))
    f.update(over)
    f["section"] = (ctypes.c_int32 * 4)(*f["section"])
    return pg.ArRotary(**f)


def _refused(rc, word):
    text = hw.lib().ar_hip_last_error().decode()
    assert rc == hw.AR_HIP_ERR_INVALID, (rc, text)
    assert word in text, text


def _ref(x):
    return ctypes.byref(x) if x is not None else None


def _grow(p, c, work=A, bytes_=1 << 20):
    return hw.lib().ar_hip_pages_grow(None, _ref(p), _ref(c), None, work, bytes_)


def _write(p, c, r, layer=0, q=A, k=A, v=A, qs=256, ks=128, heads=4, qn=None, kn=None, mode=0, out=2 * A, act=0):
    return hw.lib().ar_hip_pages_write(None, _ref(p), layer, _ref(c), q, k, v, qs, ks, heads, qn, kn, 1e-6, mode,
                                       _ref(r), out, act)


def _attend(p, c, layer=0, q=A, act=0, heads=4, out=A, work=A, bytes_=1 << 30):
    return hw.lib().ar_hip_attention_paged(None, _ref(p), layer, _ref(c), q, act, heads, out, work, bytes_)


BAD_POOLS = [(dict(k=None), "no keys"), (dict(v=A + 4), "aligned"), (dict(dtype=3), "dtype"), (dict(head_dim=96), "head_dim"),
             (dict(page_rows=48), "power of two"), (dict(page_rows=8), "power of two"), (dict(page_rows=512), "power of two"),
             (dict(layers=0), "empty"), (dict(pages=0), "empty"), (dict(pages=-1), "empty"), (dict(kv_heads=0), "empty"),
             (dict(pages=(1 << 28) + 1), "2^28"), (dict(seqs=-1), "table"), (dict(max_pages=1 << 28), "2^30")]


@pytest.mark.parametrize("over,word", BAD_POOLS)
def test_every_call_refuses_a_bad_pool(over, word):
    p, c = _pages(**over), _chunks()
    b = ctypes.c_size_t()
    L = hw.lib()
    _refused(L.ar_hip_pages_work(ctypes.byref(p), 4, ctypes.byref(b)), word)
    _refused(_grow(p, c), word)
    _refused(L.ar_hip_pages_trim(None, ctypes.byref(p), None, None, 1), word)
    _refused(L.ar_hip_pages_fork(None, ctypes.byref(p), A, A, 1, A, 1 << 20), word)
    _refused(L.ar_hip_pages_compact(None, ctypes.byref(p), None, A, 1 << 20), word)
    _refused(L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(_pages()), A, A, 1), word)
    _refused(L.ar_hip_pages_copy(None, ctypes.byref(_pages()), ctypes.byref(p), A, A, 1), word)
    _refused(_write(p, c, _rotary()), word)
    _refused(_attend(p, c), word)
    _refused(L.ar_hip_attention_paged_work(None, ctypes.byref(p), ctypes.byref(c), 4, ctypes.byref(b)), word)


def test_null_structures_and_context_are_refused():
    L, p, c, b = hw.lib(), _pages(), _chunks(), ctypes.c_size_t()
    _refused(L.ar_hip_pages_work(None, 1, ctypes.byref(b)), "null")
    _refused(L.ar_hip_pages_work(ctypes.byref(p), 1, None), "null")
    _refused(_grow(None, c), "null")
    _refused(_grow(p, None), "null")
    _refused(_attend(p, None), "null")
    _refused(_write(p, c, None), "rotary axes")
    # nothing else wrong: the context is
    other = _pages(k=1 << 40, v=1 << 41)
    for call in (lambda: _grow(p, c), lambda: _attend(p, c), lambda: _write(p, c, _rotary()),
                 lambda: L.ar_hip_pages_trim(None, ctypes.byref(p), None, None, 3),
                 lambda: L.ar_hip_pages_fork(None, ctypes.byref(p), A, A, 2, A, 1 << 20),
                 lambda: L.ar_hip_pages_compact(None, ctypes.byref(p), None, A, 1 << 20),
                 lambda: L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(other), A, A, 1),
                 lambda: L.ar_hip_attention_paged_work(None, ctypes.byref(p), ctypes.byref(c), 4, ctypes.byref(b))):
        _refused(call(), "ctx is null")


@pytest.mark.parametrize("over,word", [(dict(at=None), "cache rows"), (dict(n=0), "chunks"), (dict(n=-1), "chunks"),
                                       (dict(n=(1 << 20) + 1), "chunks"), (dict(rows=-1), "negative"),
                                       (dict(rows=(1 << 22) + 1), "2^22"),
                                       (dict(start=None, n=3, rows=2), "one row"), (dict(n=4), "sequences")])
def test_bad_chunks_are_refused(over, word):
    p, c = _pages(), _chunks(**over)
    _refused(_grow(p, c), word)
    _refused(_write(p, c, _rotary()), word)
    _refused(_attend(p, c), word)


def test_table_calls_refuse_missing_counts_entries_and_work():
    L = hw.lib()
    for p in (_pages(rows=None), _pages(refs=None)):
        _refused(_grow(p, _chunks()), "counts")
        _refused(L.ar_hip_pages_trim(None, ctypes.byref(p), None, None, 1), "counts")
        _refused(L.ar_hip_pages_fork(None, ctypes.byref(p), A, A, 1, A, 1 << 20), "counts")
    _refused(L.ar_hip_pages_compact(None, ctypes.byref(_pages(refs=None)), None, A, 1 << 20), "counts")
    _refused(_grow(_pages(table=None), _chunks()), "no table")
    p = _pages(seqs=5000)
    _refused(_grow(p, _chunks(n=4097)), "entries")
    _refused(L.ar_hip_pages_trim(None, ctypes.byref(p), A, None, 4097), "entries")
    _refused(L.ar_hip_pages_trim(None, ctypes.byref(p), A, None, -1), "entries")
    _refused(L.ar_hip_pages_trim(None, ctypes.byref(_pages()), None, None, 4), "sequences")
    _refused(L.ar_hip_pages_fork(None, ctypes.byref(p), A, A, 4097, A, 1 << 30), "entries")
    _refused(L.ar_hip_pages_fork(None, ctypes.byref(p), None, A, 1, A, 1 << 30), "null")
    _refused(L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(p), A, A, 4097), "entries")
    _refused(L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(p), A, None, 1), "null")
    b = ctypes.c_size_t()
    p = _pages()
    hw.check(L.ar_hip_pages_work(ctypes.byref(p), 2, ctypes.byref(b)))
    assert b.value > 0
    _refused(_grow(p, _chunks(), A, b.value - 1), "needed")
    _refused(_grow(p, _chunks(), None, b.value), "needed")
    _refused(_grow(p, _chunks(), A + 8, b.value), "aligned")
    _refused(L.ar_hip_pages_fork(None, ctypes.byref(p), A, A, 2, A, b.value - 1), "needed")
    _refused(L.ar_hip_pages_compact(None, ctypes.byref(p), None, A, 0), "needed")


@pytest.mark.parametrize("over", [dict(dtype=hw.DTYPE_F16), dict(layers=1), dict(kv_heads=1), dict(page_rows=32),
                                  dict(head_dim=128)])
def test_copy_refuses_pools_of_another_shape(over):
    L, p = hw.lib(), _pages()
    _refused(L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(_pages(**over)), A, A, 1), "differ")


def test_copy_refuses_pools_that_share_part_of_their_memory():
    L, p = hw.lib(), _pages()
    # (a pool array of _pages: 2 layers of 8 pages, 2 heads, 16 rows, 64 dims of fp32)
    size = p.layers * p.pages * p.kv_heads * p.page_rows * p.head_dim * 4
    big = _pages(k=1 << 40, v=(1 << 40) + 100 * size)
    for over in (dict(k=big.k + size - 16, v=big.v + 8 * size), dict(k=big.k - size + 16, v=big.v + 8 * size),
                 dict(k=big.v + 16, v=big.v + 8 * size), dict(k=big.k + 8 * size, v=big.v + size - 16),
                 dict(k=big.k - 2 * size + 16, v=big.v + 8 * size, pages=2 * big.pages)):
        _refused(L.ar_hip_pages_copy(None, ctypes.byref(big), ctypes.byref(_pages(**over)), A, A, 1), "share")
    for over, word in ((dict(v=3 * A), "share"), (dict(k=2 * A, v=A), "share"), (dict(pages=9), "two page counts")):
        _refused(L.ar_hip_pages_copy(None, ctypes.byref(p), ctypes.byref(_pages(**over)), A, A, 1), word)


@pytest.mark.parametrize("over,word", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(q=None), "both"), (dict(out=None), "both"), (dict(act=hw.DTYPE_F16), "activation dtype"), (dict(heads=3), "head counts"),
    (dict(heads=0), "head counts"), (dict(mode=2), "qk-norm"), (dict(ks=124), "kv_stride"), (dict(ks=130), "kv_stride"),
    (dict(qs=252), "q_stride"), (dict(qs=258), "q_stride"), (dict(q=A + 4), "aligned"), (dict(k=A + 8), "aligned"),
    (dict(qn=A + 4), "aligned"), (dict(out=2 * A + 8), "aligned"), (dict(out=A, act=hw.DTYPE_BF16), "in place"),
    (dict(out=A, qs=512), "in place")])
def test_write_refuses(over, word):
    _refused(_write(_pages(), _chunks(), _rotary(), **over), word)


@pytest.mark.parametrize("over,word", [
    (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(theta=float("inf")), "theta"), (dict(layout=2), "layout"), (dict(section=(16, 8, 7, 0)), "add up"),
    (dict(section=(-8, 32, 8, 0)), "section"), (dict(section=(0, 33, 0, 0)), "section"),
    (dict(layout=pg.ROPE_INTERLEAVED, section=(10, 12, 10, 0)), "interleaving"),
    (dict(axes=1, section=(31, 0, 0, 0)), "add up")])
def test_write_refuses_bad_rotary_positions(over, word):
    _refused(_write(_pages(), _chunks(), _rotary(**over)), word)


@pytest.mark.parametrize("over,word", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(act=hw.DTYPE_F16), "activation dtype"), (dict(heads=5), "head counts"), (dict(q=A + 4), "aligned"),
    (dict(out=A + 8), "aligned"), (dict(work=A + 4), "aligned")])
def test_attention_refuses(over, word):
    _refused(_attend(_pages(), _chunks(), **over), word)


def test_binding_refuses_before_the_library():
    with pytest.raises(ValueError):
        pg.Rotary(1e6, None, [8, 8, 8, 4, 4])
    with pytest.raises(ValueError):
        pg.PagedCache(None, 1, 1, 1, 64, 1, 1, dtype=hw.DTYPE_F64)


def test_calls_after_close_are_refused():
    """A closed cache hands no freed pointer on."""
    class Buf:
        def __init__(self, nbytes=0):
            self.ptr, self.nbytes, self.freed = A, nbytes, False

        def upload(self, a):
            pass

        def free(self):
            self.freed = True

    class Ctx:
        handle = None

        def __init__(self):
            self.made = []

        def allocate(self, nbytes):
            self.made.append(Buf(nbytes))
            return self.made[-1]

    ctx, given = Ctx(), Buf()
    cache = pg.PagedCache(ctx, 1, 4, 1, 64, 2, 2, v=given)
    cache._scratch(100)
    first = cache._work[-1]
    cache._scratch(90)
    assert cache._work == [first]
    cache._scratch(101)  # queued calls may use the first: it stays
    assert not first.freed and cache._work[-1].nbytes >= 200
    at = Buf()
    ch = pg.Chunks(1, 1, at=at)
    cache.close()
    assert all(b.freed for b in ctx.made) and not given.freed
    for call in (lambda: cache.grow(ch), lambda: cache.trim(None, None, 1), lambda: cache.attention(0, ch, at, at, 1),
                 lambda: cache.compact(), lambda: cache.copy(cache, at, at, 1)):
        with pytest.raises(Exception, match="no keys"):
            call()


def test_copy_to_a_cache_of_another_context(monkeypatch):
    """On one device it is ordered with both contexts' work; on another device it is refused before the library."""
    class Buf:
        ptr = A

    class Ctx:
        def __init__(self, name, index):
            self.name, self.index, self.handle = name, index, A

        def synchronize(self):
            done.append(self.name)

    class Lib:
        def ar_hip_pages_copy(self, *args):
            done.append("copy")
            return hw.AR_HIP_OK

    done = []
    monkeypatch.setattr(pg, "lib", Lib)
    a, b, c = (pg.PagedCache(x, 1, 4, 1, 64, 1, 1, k=Buf, v=Buf, table=Buf, rows=Buf, refs=Buf)
               for x in (Ctx("a", 0), Ctx("b", 0), Ctx("c", 1)))
    a.copy(a, Buf, Buf, 1)
    assert done == ["copy"]
    done.clear()
    a.copy(b, Buf, Buf, 1)
    assert done == ["b", "copy", "a"]
    done.clear()
    with pytest.raises(ValueError, match="device"):
        a.copy(c, Buf, Buf, 1)
    assert not done


def test_a_cache_keeps_few_work_sizes(monkeypatch):
    """A server's row counts differ in every step: what the cache keeps of them has an end, and sizes stay right."""
    class Buf:
        ptr, nbytes = A, 1 << 40

    class Ctx:
        handle = A

    class Lib:
        def ar_hip_attention_paged_work(self, ctx, pages, chunks, heads, out):
            asked.append(chunks._obj.rows)
            out._obj.value = 1000 + chunks._obj.rows
            return hw.AR_HIP_OK

        def ar_hip_pages_work(self, pages, n, out):
            out._obj.value = 10 + n
            return hw.AR_HIP_OK

        def ar_hip_attention_paged(self, *args):
            return hw.AR_HIP_OK

    asked, needed = [], []
    monkeypatch.setattr(pg, "lib", Lib)
    cache = pg.PagedCache(Ctx(), 1, 4, 1, 64, 1, 1, k=Buf, v=Buf, table=Buf, rows=Buf, refs=Buf)
    cache._work.append(Buf)
    monkeypatch.setattr(cache, "_scratch", lambda need: needed.append(need) or Buf)
    for rows in list(range(1, 500)) + [499, 1]:
        cache.attention(0, pg.Chunks(1, rows, at=Buf, start=Buf), Buf, Buf, 1)
        assert needed[-1] == 1000 + rows and len(cache._need) <= 64
        cache._table_scratch(rows)
        assert needed[-1] == 10 + rows and len(cache._need) <= 64
    assert asked == list(range(1, 500)) + [1]


@pytest.mark.parametrize("room", range(5))
def test_a_cache_that_does_not_fit_leaves_nothing_behind(room):
    """Whichever of its buffers cannot be had, those before it are given back."""
    class Buf:
        ptr, freed = A, False

        def upload(self, a):
            pass

        def free(self):
            self.freed = True

    class Ctx:
        def __init__(self):
            self.made = []

        def allocate(self, nbytes):
            if len(self.made) == room:
                raise hw.HardwareException(1, "out of memory")
            self.made.append(Buf())
            return self.made[-1]

    ctx = Ctx()
    with pytest.raises(hw.HardwareException, match="out of memory"):
        pg.PagedCache(ctx, 1, 4, 1, 64, 2, 2)
    assert len(ctx.made) == room and all(b.freed for b in ctx.made)
