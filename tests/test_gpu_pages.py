"""The page operators against a model that does one thing after another on host
lists; every table, count, length and byte of the pools is equal after each
call.  Then the operators together, as a server uses them."""
import ctypes

import numpy as np
import pytest

from gpu_util import D, H, banner, p
from paged_util import Cache, angles, grid, ints, normal, rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


class Paged(Cache):
    """A cache whose calls are made on the device and, by definition, on the model."""

    def need(self, n):
        return -(-n // self.page)

    def free_pages(self):
        return [i for i in range(self.pages) if self.refs[i] == 0]

    def work(self):
        if not hasattr(self, "ws"):
            self.ws = D(np.random.default_rng(0).integers(0, 256, self.lib.gsdh_pages_workspace_bytes(self.at)).astype(np.uint8))
        return self.ws

    def take(self, seqs, counts):
        a, b = ints(seqs), ints(counts)
        self.lib.gsdh_pages_take(None, self.at, p(a), p(b), len(seqs))
        bits, seen, free, used = 0, set(), self.free_pages(), 0
        for s, k in zip(seqs, counts):
            if not 0 <= s < self.seqs or k < 0:
                bits |= 1
                seen.add(s)   # (the first place that names a sequence counts, whatever it asks)
                continue
            if s in seen:
                bits |= 8
                continue
            seen.add(s)
            n = int(self.lens[s])
            if n + k > self.width * self.page:
                bits |= 1
                continue
            m = self.need(n + k) - self.need(n)
            if m and used + m > len(free):
                bits |= 2
                used += m
                continue
            for j in range(m):
                self.tables[s, self.need(n) + j] = free[used + j]
                self.refs[free[used + j]] = 1
            used += m
            self.lens[s] += k
        return bits

    def fork(self, src, dst):
        a, b = ints(src), ints(dst)
        self.lib.gsdh_pages_fork(None, self.at, p(a), p(b), len(src), p(self.work()), self.work().nbytes)
        bits, seen, free, used, before = 0, set(), self.free_pages(), 0, self.lens.copy()
        for s, d in zip(src, dst):
            if not 0 <= s < self.seqs or not 0 <= d < self.seqs:
                bits |= 1
                if 0 <= d < self.seqs:
                    seen.add(d)
                continue
            if d in seen or before[d]:
                seen.add(d)
                bits |= 8
                continue
            seen.add(d)
            n = int(before[s])
            full, part = divmod(n, self.page)
            if part:
                used += 1
                if used > len(free):
                    bits |= 2
                    continue
                new, old = free[used - 1], self.tables[s, full]
                self.refs[new] = 1
                for pool in (self.k, self.v):
                    at = (slice(None), new, slice(None), slice(0, part)) if self.head_major else (slice(None), new, slice(0, part))
                    pool[at] = pool[(slice(None), old) + at[2:]]
                self.tables[d, full] = new
            self.tables[d, :full] = self.tables[s, :full]
            np.add.at(self.refs, self.tables[s, :full], 1)
            self.lens[d] = n
        return bits

    def free(self, seqs):
        a = ints(seqs)
        self.lib.gsdh_pages_free(None, self.at, p(a), len(seqs))
        bits = 0
        for s in seqs:
            if not 0 <= s < self.seqs:
                bits |= 1
                continue
            k = self.need(int(self.lens[s]))
            np.add.at(self.refs, self.tables[s, :k], -1)
            self.tables[s, :k] = -1
            self.lens[s] = 0
        return bits

    def compact(self):
        n = D(np.full(1, -5, np.int32))
        self.lib.gsdh_pages_compact(None, self.at, p(n), p(self.work()), self.work().nbytes)
        used = int((self.refs > 0).sum())
        holes = [i for i in range(used) if self.refs[i] == 0]
        for a, b in zip([i for i in range(used, self.pages) if self.refs[i] > 0], holes):
            for pool in (self.k, self.v):
                pool[:, b] = pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.tables[self.tables == a] = b
        assert H(n, np.int32, 1)[0] == used
        return 0

    def copy(self, src, dst):
        a, b = ints(src), ints(dst)
        self.lib.gsdh_pages_copy(None, self.at, p(a), p(b), len(src), p(self.work()), self.work().nbytes)
        ok = lambda x: 0 <= x < self.pages  # noqa: E731
        bits, old, seen = 0, (self.k.copy(), self.v.copy()), set()
        targets = {d for s, d in zip(src, dst) if ok(s) and ok(d)}
        for s, d in zip(src, dst):
            if s < 0 or d < 0:
                continue
            if not (ok(s) and ok(d)):
                bits |= 1
            elif d in seen or s in targets:
                bits |= 8
                seen.add(d)
            else:
                seen.add(d)
                for pool, was in zip((self.k, self.v), old):
                    pool[:, d] = was[:, s]
        return bits

    def same(self, bits=0):
        for name in ("refs", "lens", "tables", "k", "v"):
            assert np.array_equal(self.download(name), getattr(self, name)), name
        assert self.status() == bits
        if bits:
            self.clear_status()
        # every page is held as often as tables name it
        count = np.zeros(self.pages, np.int32)
        for s in range(self.seqs):
            np.add.at(count, self.tables[s, :self.need(int(self.lens[s]))], 1)
        assert np.array_equal(count, self.refs)


def _cache(kind="f16", layers=3, pages=60, page=8, kv=2, hd=64, head_major=False, seqs=12, width=10, lens=(), seed=1):
    c = Paged(kind, layers, pages, page, kv, hd, head_major, seqs, width)
    return c.fill(list(lens), np.random.default_rng(seed), normal)


@pytest.mark.parametrize("kind,head_major,page,kv,hd", [("f16", False, 8, 2, 64), ("e4m3", True, 16, 1, 64), ("bf16", True, 8, 3, 128),
                                                        ("e4m3", False, 32, 2, 256)])
def test_each(lib, kind, head_major, page, kv, hd):
    banner(f"pages {kind} page {page} {kv}x{hd} {'head' if head_major else 'slot'}")
    c = _cache(kind, 3, 80, page, kv, hd, head_major, 12, 10, [3 * page, page + 3, 1, 2 * page + 1, 0, 5 * page - 1])
    c.same()
    bits = c.take([0, 2, 4, 1], [1, page, 2 * page + 1, 0])
    c.same(bits)
    bits = c.fork([0, 0, 1, 2, 3], [6, 7, 8, 9, 10])
    c.same(bits)
    bits = c.free([0, 8, 5, 11])
    c.same(bits)
    c.compact()
    c.same()
    c.compact()   # (nothing left to move)
    c.same()
    last = c.pages - 1
    bits = c.copy([0, 1, -1, 2, 0], [last, last - 1, 3, -1, last - 2])
    c.same(bits)


def test_lists_that_name_things_twice_or_wrongly(lib):
    banner("pages: duplicates, wrong indices, too few pages")
    c = _cache(pages=20, lens=[16, 9, 20, 0, 0, 1], seqs=9)
    c.same(c.take([1, 1, 9, -1, 2, 3], [8, 80, 1, 1, -1, 3]))
    c.same(c.take([0], [65]))            # beyond the table
    c.same(c.take([3, 0, 4, 1, 5], [40, 64, 200, 30, 7]))   # the second does not fit, the table ends before the third's
    c.same(c.fork([0, 1, 2, 5, 5, 9, 0], [6, 6, 1, 7, 7, 8, -2]))
    c.same(c.free([0, 0, 6, 9, 8]))
    c.same(c.free([0]))
    c.same(c.fork([8, 8], [3, 4]) if c.lens[3] == 0 else c.fork([8], [4]))   # a fork of nothing
    c.same(c.fork([4], [4]))
    c.same(c.copy([1, 2, 1, 3, 20, 0], [0, 0, 5, 1, 4, 20]))
    c.compact()
    c.same()


def test_exhausted_pool_gives_pages_back(lib):
    """The sequence that takes the last pages and still lacks some keeps none of them."""
    banner("pages: an exhausted pool")
    c = _cache(pages=9, lens=[8, 8, 8], seqs=9, width=16)
    assert c.take([3, 4, 5], [24, 32, 8]) == 2       # 3 pages, then 4 of the 3 left, then none counted
    c.same(2)
    assert c.take([4], [24]) == 0
    c.same()
    assert c.take([5, 0], [1, 1]) == 2
    c.same(2)
    c.lens[2] -= 3
    c.upload()
    assert c.fork([2, 2], [5, 6]) == 2   # partly filled: a page each, none left
    c.same(2)
    c.lens[2] += 3
    c.upload()
    assert c.fork([2, 2], [5, 6]) == 0   # full: shared
    c.same()


def test_corrupt_state_is_not_followed(lib):
    """Tables that name pages outside the pool, or pages that nobody holds: no
    byte outside the pool is touched, the status word tells."""
    banner("pages: corrupt tables")
    c = _cache(pages=20, lens=[16, 9, 20, 12], seqs=6, layers=1)
    free = c.free_pages()[-1]
    c.tables[0, 1], c.tables[1, 0], c.tables[2, 2] = 20, -9, free
    c.upload()
    c.lib.gsdh_pages_compact(None, c.at, None, p(c.work()), c.work().nbytes)
    assert c.status() == 1
    c.clear_status()
    c.upload()
    a, b = ints([0, 1, 2]), ints([4, 5, 4])
    c.lib.gsdh_pages_fork(None, c.at, p(a), p(b), 3, p(c.work()), c.work().nbytes)
    assert c.status() & 1
    c.clear_status()
    c.upload()
    c.lib.gsdh_pages_free(None, c.at, p(a), 3)
    assert c.status() == 1
    assert (c.download("refs") >= 0).all()
    assert (c.download("lens")[:3] == 0).all()


@pytest.mark.parametrize("pages", [1, 63, 64, 1023, 1024, 1025, 8191, 8192, 8193, 20000])
def test_pool_sizes(lib, pages):
    """Order and counts over every size of a step of the scan."""
    banner(f"pages: a pool of {pages}")
    rng = np.random.default_rng(pages)
    c = Paged("e4m3", 1, pages, 8, 1, 64, False, 40, max(1, pages // 4) + 1)
    held = rng.random(pages) < 0.5
    cuts = np.array_split(rng.permutation(np.flatnonzero(held)), 20)
    for s, part in enumerate(cuts):
        k = min(len(part), c.width)
        c.tables[s, :k], c.lens[s] = part[:k], 8 * k
        c.refs[part[:k]] = 1
    c.k[:] = rng.integers(0, 120, c.k.shape)
    c.v[:] = rng.integers(0, 120, c.v.shape)
    c.upload()
    c.same()
    c.same(c.take(list(range(20, 40)), [int(x) for x in rng.integers(0, max(2, 8 * pages // 60), 20)]))
    c.same(c.free(list(range(0, 40, 3))))
    c.compact()
    c.same()


def test_random_calls(lib):
    """A hundred calls in a row, lists with duplicates and wrong indices among them."""
    banner("pages: a hundred random calls")
    rng = np.random.default_rng(42)
    c = _cache("e4m3", 2, 70, 8, 1, 64, True, 16, 9, [5, 70, 0, 33, 8])
    for _ in range(100):
        n = int(rng.integers(1, 9))
        some = [int(x) for x in rng.integers(-1, 17, n)]
        op = rng.integers(0, 6)
        if op <= 1:
            bits = c.take(some, [int(x) for x in rng.integers(-1, 30, n)])
        elif op == 2:
            bits = c.fork(some, [int(x) for x in rng.integers(-1, 17, n)])
        elif op == 3:
            bits = c.free(some)
        elif op == 4:
            bits = c.compact()
        else:
            free = c.free_pages()
            bits = c.copy([int(x) for x in rng.integers(-1, 71, n)], [int(x) for x in rng.choice(free + [-1], n)])
        c.same(bits)


def test_largest_lists(lib):
    """8192 sequences, all of them in one list."""
    banner("pages: 8192 sequences")
    c = Paged("e4m3", 1, 9000, 8, 1, 64, False, 8192, 2)
    c.k[:], c.v[:] = 1, 2
    c.upload()
    rng = np.random.default_rng(4)
    c.same(c.take([int(x) for x in rng.permutation(8192)], [int(x) for x in rng.integers(0, 12, 8192)]))
    c.same(c.free([int(x) for x in rng.permutation(8192)[:5000]]))
    c.compact()
    c.same()


def test_long_lists_with_faults(lib):
    """Lists longer than a planning block's threads: repeats, counts below
    zero and indices outside in every part of them, forks of partly filled pages."""
    banner("pages: lists of thousands with faults in them")
    c = Paged("e4m3", 1, 9000, 8, 1, 64, False, 4000, 4)
    c.k[:], c.v[:] = 1, 2
    c.upload()
    rng = np.random.default_rng(5)
    seqs, counts = rng.integers(-2, 2002, 3500), rng.integers(-1, 12, 3500)
    c.same(c.take([int(x) for x in seqs], [int(x) for x in counts]))
    c.same(c.take([2, 2], [-1, 3]))   # the first place counts, whatever it asks
    held = np.flatnonzero(c.lens)
    assert len(held) > 1100 and (c.lens[held] % 8 != 0).sum() > 1000
    src, dst = rng.choice(held, 3000), rng.integers(1990, 4002, 3000)
    c.same(c.fork([int(x) for x in src], [int(x) for x in dst]))
    c.same(c.free([int(x) for x in rng.integers(0, 4001, 2500)]))
    c.compact()
    c.same()


def test_wants_beyond_32_bits(lib):
    """Sequences that together want more pages than 32 bits count: the first
    takes the whole pool of 2^20, the others stay as they were."""
    banner("pages: 2100 sequences that want 2^20 pages each")
    n, pages = 2100, 1 << 20
    small = Paged("f16", 1, 8, 8, 1, 64, False, 1, 1)   # (its rows are not touched)
    tables = ctypes.c_void_p()
    lib.gsdh_malloc(ctypes.byref(tables), 4 * n * pages)
    refs, lens = ints(np.zeros(pages, np.int32)), ints(np.zeros(n, np.int32))
    c = small.struct(refs=refs.ptr, lens=lens.ptr, tables=tables.value, n_pages=pages, n_seqs=n, table_width=pages)
    seqs, counts = ints(np.arange(n)), ints(np.full(n, 8 * pages))
    lib.gsdh_pages_take(None, ctypes.byref(c), p(seqs), p(counts), n)
    assert H(lens, np.int32, n).tolist() == [8 * pages] + [0] * (n - 1)
    assert (H(refs, np.int32, pages) == 1).all() and small.status() == 2
    row = np.empty(pages, np.int32)
    lib.gsdh_memcpy_d2h(row.ctypes.data_as(ctypes.c_void_p), tables, row.nbytes, None)
    lib.gsdh_stream_sync(None)
    assert np.array_equal(row, np.arange(pages))
    lib.gsdh_free(tables)


def test_serving(lib):
    """The operators as a server runs them: prompts stored, decode steps of a
    changing batch (take, store, attend), forks, ends, compactions; every
    step's attention against the definition over what each sequence was given."""
    banner("pages: a server's steps")
    rng = np.random.default_rng(7)
    heads, kv, hd, scale = 8, 2, 64, 0.125
    c = Paged("f16", 2, 40, 8, kv, hd, False, 8, 12)
    table = angles(96, hd)
    da = D(table)
    active = []

    def step(seqs, pos):
        """One layer after another: rows of new tokens stored; the rotated q of each."""
        out = []
        for layer in range(2):
            x = grid(rng, (len(seqs), heads + 2 * kv, hd))
            dx, q, ds, dp = D(x), D(np.zeros((len(seqs), heads, hd), np.float32)), ints(seqs), ints(pos)
            at = lambda h: ctypes.c_void_p(dx.ptr.value + 4 * h * hd)  # noqa: E731
            w = (heads + 2 * kv) * hd
            c.lib.gsdh_paged_rope_store(None, c.at, layer, at(0), w, at(heads), w, at(heads + kv), w, p(q), heads * hd, p(ds), p(dp),
                                        len(seqs), heads, p(da), 96, 1)
            k = rotate(x[:, heads:heads + kv], table[pos], 1)
            for t, (s, n) in enumerate(zip(seqs, pos)):
                c.set_values(0, layer, s, [n], k[t:t + 1])
                c.set_values(1, layer, s, [n], x[t:t + 1, heads + kv:])
            out.append(H(q, np.float32, len(seqs) * heads * hd).reshape(-1, heads, hd))
        return out

    ws = c.space(8, heads)
    for i in range(30):
        empty = [s for s in range(8) if c.lens[s] == 0]
        if i % 3 == 0 and empty and len(c.free_pages()) > 6:   # a prompt comes
            s, n = empty[0], int(rng.integers(1, 30))
            assert c.take([s], [n]) == 0
            step([s] * n, list(range(n)))
            active.append(s)
        elif i % 7 == 4 and active and len(empty) > 1 and len(c.free_pages()) > 8:
            src = active[int(rng.integers(len(active)))]
            assert c.fork([src, src], empty[:2]) == 0
            active += empty[:2]
        elif i % 5 == 3 and len(active) > 2:
            gone = [active.pop(int(rng.integers(len(active)))) for _ in range(2)]
            assert c.free(gone) == 0
            c.compact()
        if not active or len(c.free_pages()) < len(active):
            continue
        active = [s for s in active if c.lens[s] < 95]
        assert c.take(active, [1] * len(active)) == 0
        qs = step(active, [int(c.lens[s]) - 1 for s in active])
        for layer, q in enumerate(qs):
            got = c.run_attend(layer, q, active, scale, ws=ws)
            want, mag, top, dot = c.attend(layer, q, active, np.float32(scale))
            # (the bound of the attention's own tests)
            eps = 2 * ((hd + 16) * dot + 8 * top) + 96 / 128 + 96
            assert (np.abs(got - want) <= 2.0 ** -24 * eps[..., None] * mag).all()
    c.same()
    assert len(active) > 2


def test_captured(lib):
    """take, fork, free and compact in one graph, replayed on new lists and states."""
    banner("pages: a captured sequence of calls")
    c = _cache(pages=50, lens=[20, 9, 30, 5], seqs=12)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(stream))
    lists = {n: ints([0, 0]) for n in ("take", "count", "src", "dst", "gone")}
    c.work()
    n_used = ints([0])

    def put(buf, a):
        a = np.asarray(a, np.int32)
        lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
        lib.gsdh_stream_sync(None)

    lib.gsdh_stream_begin_capture(stream)
    lib.gsdh_pages_take(stream, c.at, p(lists["take"]), p(lists["count"]), 2)
    lib.gsdh_pages_fork(stream, c.at, p(lists["src"]), p(lists["dst"]), 2, p(c.ws), c.ws.nbytes)
    lib.gsdh_pages_free(stream, c.at, p(lists["gone"]), 2)
    lib.gsdh_pages_compact(stream, c.at, p(n_used), p(c.ws), c.ws.nbytes)
    lib.gsdh_stream_end_capture(stream, ctypes.byref(graph))
    for values in (dict(take=[0, 3], count=[3, 11], src=[0, 1], dst=[4, 5], gone=[1, 6]),
                   dict(take=[4, 5], count=[1, 1], src=[3, 3], dst=[6, 7], gone=[0, 2]),
                   dict(take=[8, 6], count=[40, 2], src=[8, 5], dst=[9, 10], gone=[3, 4])):
        for k, v in values.items():
            put(lists[k], v)
        lib.gsdh_graph_replay(graph, stream)
        lib.gsdh_stream_sync(stream)
        got = {n: c.download(n) for n in ("refs", "lens", "tables", "k", "v")}
        # the model's turn: its own eager calls run on a second cache of the same state
        twin = Paged.__new__(Paged)
        twin.__dict__.update({k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in c.__dict__.items() if k != "ws"})
        twin.upload()
        assert twin.take(values["take"], values["count"]) == 0
        twin.same(0)
        assert twin.fork(values["src"], values["dst"]) == 0
        twin.same(0)
        twin.free(values["gone"])
        twin.compact()
        twin.same(0)
        for n, a in got.items():
            assert np.array_equal(a, getattr(twin, n)), n
            setattr(c, n, getattr(twin, n))
    lib.gsdh_graph_destroy(graph)
    lib.gsdh_stream_destroy(stream)


def test_forks_of_bad_tables_are_left_out(lib):
    """A source whose table names a page outside the pool, wherever in it: the
    entry leaves everything as it was, and keeps no page; the others are done."""
    banner("pages: forks of tables with bad pages")
    lens = [20, 9, 1200, 1200, 24, 700, 16]
    c = _cache(pages=500, lens=lens, seqs=20, width=160, layers=1)
    bad = {0: (0, 500), 2: (149, -1), 3: (70, 1 << 30), 4: (2, -9), 6: (1, 500)}
    for s, (j, page) in bad.items():
        c.tables[s, j] = page
    c.upload()
    src, dst = [0, 1, 2, 3, 5, 4, 6, 1, 0, 5, 2], [8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18]
    a, b = ints(src), ints(dst)
    c.lib.gsdh_pages_fork(None, c.at, p(a), p(b), len(src), p(c.work()), c.work().nbytes)
    free, back = iter(c.free_pages()), []
    for s, d in zip(src, dst):
        if s in bad:
            if lens[s] % c.page:
                back.append(next(free))   # (dealt out and given back: its rows may be any)
            continue
        full, part = divmod(lens[s], c.page)
        c.tables[d, :full] = c.tables[s, :full]
        np.add.at(c.refs, c.tables[s, :full], 1)
        c.lens[d] = lens[s]
        if part:
            new, old = next(free), c.tables[s, full]
            c.tables[d, full], c.refs[new] = new, 1
            for pool in (c.k, c.v):
                pool[:, new, :part] = pool[:, old, :part]
    for name in ("refs", "lens", "tables"):
        assert np.array_equal(c.download(name), getattr(c, name)), name
    for name in ("k", "v"):
        assert np.array_equal(np.delete(c.download(name), back, 1), np.delete(getattr(c, name), back, 1)), name
    assert len(back) == 2 and c.status() == 1


def test_long_lists_of_forks_of_bad_tables(lib):
    """The same beyond a planning block's threads: a bad source in every part of the list, often."""
    banner("pages: 3000 forks, some of tables with bad pages")
    c = Paged("e4m3", 1, 5000, 8, 1, 64, False, 4000, 4)
    c.k[:], c.v[:] = 1, 2
    rng = np.random.default_rng(8)
    c.tables[:1000] = rng.permutation(5000)[:4000].reshape(1000, 4)
    c.refs[c.tables[:1000].reshape(-1)] = 1
    c.lens[:1000] = rng.integers(25, 33, 1000)
    bad = rng.choice(1000, 200, replace=False)
    c.tables[bad, rng.integers(0, 3, 200)] = 5000
    c.upload()
    src, dst = rng.integers(0, 1000, 3000), 1000 + np.arange(3000)
    a, b = ints(src), ints(dst)
    c.lib.gsdh_pages_fork(None, c.at, p(a), p(b), 3000, p(c.work()), c.work().nbytes)
    good = ~np.isin(src, bad)
    out = np.flatnonzero(c.lens[src] < 32)[1000:]   # (a page of its own for each: the first thousand have one)
    done = good.copy()
    done[out] = False
    refs, tables, got = c.download("refs"), c.download("tables"), c.download("lens")
    assert np.array_equal(got[1000:], np.where(done, c.lens[src], 0))
    assert (tables[1000:][~done] == -1).all() and np.array_equal(tables[:1000], c.tables[:1000])
    assert np.array_equal(tables[1000:][done][:, :3], c.tables[src[done], :3])
    count = np.zeros(5000, np.int32)
    held = np.concatenate([c.tables[:1000].reshape(-1), tables[1000:][done].reshape(-1)])
    np.add.at(count, held[(held >= 0) & (held < 5000)], 1)
    names = np.zeros(5000, bool)   # (the pages that the bad entries' places held stay held)
    names[np.flatnonzero((c.refs == 1) & (count == 0))] = True
    assert np.array_equal(refs, count + names)
    assert len(out) and c.status() == 3


def test_free_of_a_bad_length(lib):
    """A sequence whose length no table can hold stays as it was, pages and all, however often it is listed."""
    banner("pages: free of lengths outside the tables")
    c = _cache(pages=40, lens=[16, 9, 20, 12], seqs=6, layers=1)
    good = c.lens.copy()
    c.lens[1], c.lens[2] = 8 * 10 + 1, -3
    c.upload()
    a = ints([1, 2, 0, 1, 2])
    c.lib.gsdh_pages_free(None, c.at, p(a), 5)
    c.refs[c.tables[0, :2]] = 0
    c.tables[0, :2], c.lens[0], good[0] = -1, 0, 0
    for name in ("refs", "lens", "tables"):
        assert np.array_equal(c.download(name), getattr(c, name)), name
    assert c.status() == 1
    # with its length put right it gives its pages back
    c.lens[:] = good
    c.upload()
    c.same(c.free([1, 2]))


def test_a_padded_step(lib):
    """One captured step of up to five rows, replayed for fewer: the list of take
    names every sequence, with a count of 0 where none is wanted, the rows of
    store and attention are padded with -1, a list of sequences that ended with
    one that is free.  No bit of the status word is raised."""
    banner("pages: a padded step, captured")
    rng = np.random.default_rng(17)
    heads, kv, hd, rows, scale = 8, 2, 64, 5, 0.125
    c = _cache("f16", 1, 40, 8, kv, hd, False, 7, 8, [7, 8, 30, 0, 0, 1, 0])
    table = angles(64, hd)
    da, w = D(table), (heads + 2 * kv) * hd
    every, counts, ended = ints(range(7)), ints([0] * 7), ints([6] * 2)
    seqs, pos = ints([-1] * rows), ints([0] * rows)
    dx, q, out = D(np.zeros((rows, w), np.float32)), D(np.zeros((rows, heads, hd), np.float32)), D(np.zeros((rows, heads, hd), np.float32))
    at = lambda h: ctypes.c_void_p(dx.ptr.value + 4 * h * hd)  # noqa: E731
    ws, stream, graph = c.space(rows, heads), ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(stream))

    def put(buf, a, dtype=np.int32):
        a = np.ascontiguousarray(a, dtype)
        lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
        lib.gsdh_stream_sync(None)

    lib.gsdh_stream_begin_capture(stream)
    lib.gsdh_pages_free(stream, c.at, p(ended), 2)
    lib.gsdh_pages_take(stream, c.at, p(every), p(counts), 7)
    lib.gsdh_paged_rope_store(stream, c.at, 0, at(0), w, at(heads), w, at(heads + kv), w, p(q), heads * hd, p(seqs), p(pos), rows, heads,
                              p(da), 64, 1)
    lib.gsdh_paged_attention(stream, c.at, 0, p(q), heads * hd, p(seqs), rows, heads, scale, 0, p(out), heads * hd, p(ws), ws.nbytes)
    lib.gsdh_stream_end_capture(stream, ctypes.byref(graph))
    for active, gone in (([0, 2, 5], [6, 6]), ([1, 0, 2, 5, 3], [6, 6]), ([3], [2, 6]), ([3, 0], [0, 1]), ([], [6, 4])):
        x = grid(rng, (rows, heads + 2 * kv, hd))
        put(ended, gone)
        put(counts, [int(s in active) for s in range(7)])
        # (the sequence that ends and is active starts again)
        where = [0 if s in gone else int(c.lens[s]) for s in active]
        put(seqs, active + [-1] * (rows - len(active)))
        put(pos, where + [0] * (rows - len(active)))
        put(dx, x.reshape(rows, w), np.float32)
        lib.gsdh_memcpy_h2d(out.ptr, np.full(rows * heads * hd, 7, np.float32).ctypes.data_as(ctypes.c_void_p), 4 * rows * heads * hd, None)
        lib.gsdh_graph_replay(graph, stream)
        lib.gsdh_stream_sync(stream)
        # the same on the model
        for s in set(gone):
            k = c.need(int(c.lens[s]))
            np.add.at(c.refs, c.tables[s, :k], -1)
            c.tables[s, :k], c.lens[s] = -1, 0
        for s in sorted(active):
            if c.lens[s] % c.page == 0:
                new = c.free_pages()[0]
                c.tables[s, c.lens[s] // c.page], c.refs[new] = new, 1
            c.lens[s] += 1
        rot = rotate(x[:len(active), heads:heads + kv], table[where], 1)
        for t, (s, n) in enumerate(zip(active, where)):
            c.set_values(0, 0, s, [n], rot[t:t + 1])
            c.set_values(1, 0, s, [n], x[t:t + 1, heads + kv:])
        c.same(0)
        got = H(out, np.float32, rows * heads * hd).reshape(rows, heads, hd)
        assert (got[len(active):] == 7).all()
        if active:
            qs = rotate(x[:len(active), :heads], table[where], 1)
            want, mag, top, dot = c.attend(0, qs, active, np.float32(scale))
            eps = 2 * ((hd + 16) * dot + 8 * top) + 64 / 128 + 96   # (the bound of the attention's own tests)
            assert (np.abs(got[:len(active)] - want) <= 2.0 ** -24 * eps[..., None] * mag).all()
    lib.gsdh_graph_destroy(graph)
    lib.gsdh_stream_destroy(stream)
