"""gsdh_paged_attention against softmax(q K) V in 64 bits over the rows that a
sequence's table names.

Tolerances, per output element, in units of sum P |V| (what the products
add up): a score s = scale * sum q k is off by at most (hd + 16) half steps of
fp32 of scale * sum |q k| (its accumulation, the split of q; nothing where the
products are exact) and 8 steps of |s| (its scaling and the exponential), so P
is off by twice that; the sum over n positions is accumulated 32 at a time, in
four waves and a join, (n / 128 + 96) steps deep."""
import ctypes

import numpy as np
import pytest

from gpu_util import D, H, banner, p
from paged_util import Cache, encode, grid, ints, nan_bits, normal

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def check(got, want, mag, top, dot, lens, exact_dots=False):
    for i, n in enumerate(lens):
        if np.isnan(want[i]).all():
            continue
        eps = 2 * ((0 if exact_dots else got.shape[2] + 16) * dot[i] + 8 * top[i]) + n / 128 + 96
        bound = STEP * eps[:, None] * mag[i] + 1e-30
        assert np.isfinite(got[i]).all(), i
        off = np.abs(got[i] - want[i]) / bound
        assert off.max() <= 1, (i, n, off.max())


LENS = [0, 1, 2, 31, 32, 33, 127, 128, 129, 160, 300]


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (8, 2, 128), (4, 4, 128), (6, 2, 64), (16, 2, 256), (16, 1, 128), (1, 1, 64)])
@pytest.mark.parametrize("page,head_major", [(8, False), (16, True), (128, False)])
def test_ragged_batch(lib, kind, heads, kv, hd, page, head_major):
    """Every length, an idle row, padding; NaN wherever nobody wrote; padded strides."""
    banner(f"paged attention {kind} {heads}/{kv}x{hd} page {page} {'head' if head_major else 'slot'}")
    rng = np.random.default_rng(heads * hd + page)
    c = Cache(kind, 2, sum(-(-n // page) for n in LENS) + 5, page, kv, hd, head_major, len(LENS), 300 // page + 2).fill(LENS, rng, grid)
    seqs = [3, -1, 10, 0, 9, 8, 7, 7, 6, 5, 4, 2, 1, -1]
    q, scale = grid(rng, (len(seqs), heads, hd)), 1.0 / float(np.sqrt(hd))
    got = c.run_attend(1, q, seqs, scale, q_pad=8, out_pad=12)
    want = c.attend(1, q, seqs, scale)
    check(got, *want, [c.lens[s] if s >= 0 else 0 for s in seqs], exact_dots=True)
    for i, s in enumerate(seqs):
        if s < 0:
            assert (got[i] == 7.0).all()
        elif c.lens[s] == 0:
            assert (got[i] == 0).all()
    assert c.status() == 0


@pytest.mark.parametrize("kind,hd,window", [("f16", 128, 1), ("bf16", 64, 31), ("e4m3", 128, 32), ("f16", 64, 100), ("e4m3", 256, 129),
                                            ("bf16", 128, 100000)])
def test_window(lib, kind, hd, window):
    banner(f"paged attention {kind} hd {hd} window {window}")
    rng = np.random.default_rng(window)
    lens = LENS + [1000]
    c = Cache(kind, 1, 200, 16, 2, hd, False, len(lens), 64).fill(lens, rng, grid)
    # the rows that the window leaves behind may hold anything
    for s, n in enumerate(lens):
        gone = np.arange(max(0, n - window))
        if len(gone):
            for pool in (c.k, c.v):
                pool[c.rows(None, 0, gone, c.tables[s])] = nan_bits((len(gone), 2, hd), kind)
    c.upload()
    q = grid(rng, (len(lens), 8, hd))
    got = c.run_attend(0, q, range(len(lens)), 0.11, window, identity=True)
    check(got, *c.attend(0, q, range(len(lens)), np.float32(0.11), window), [min(n, window) for n in lens], exact_dots=True)


@pytest.mark.parametrize("kind,heads,kv,hd,n", [("f16", 32, 8, 128, 8192), ("bf16", 8, 2, 128, 30011), ("e4m3", 16, 2, 64, 12345),
                                                ("f16", 4, 1, 256, 9001)])
def test_long_split_and_joined(lib, kind, heads, kv, hd, n):
    """Rows split over many blocks beside short ones, any values, the same bits twice."""
    banner(f"paged attention {kind} {heads}/{kv}x{hd} over {n}")
    rng = np.random.default_rng(n)
    lens = [n, 5, n // 3, 0]
    c = Cache(kind, 1, sum(-(-x // 64) for x in lens), 64, kv, hd, True, 4, -(-n // 64)).fill(lens, rng, normal)
    q, scale = 1.5 * normal(rng, (4, heads, hd)), 1.0 / float(np.sqrt(hd))
    ws = c.space(4, heads)
    got = c.run_attend(0, q, [2, 0, 1, 3], scale, ws=ws)
    check(got, *c.attend(0, q, [2, 0, 1, 3], np.float32(scale)), [c.lens[s] for s in (2, 0, 1, 3)])
    for _ in range(3):
        assert np.array_equal(got, c.run_attend(0, q, [2, 0, 1, 3], scale, ws=ws))
    # a row's result stands for itself: alone, and beside others
    one = c.run_attend(0, q[1:2], [0], scale, ws=ws)
    check(one, *c.attend(0, q[1:2], [0], np.float32(scale)), [n])


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
def test_every_position_counts(lib, kind):
    """One position that outweighs all others (its score 40 above theirs), at
    every edge of tiles, pages and splits: the output is its V row."""
    rng = np.random.default_rng(3)
    n, hd = 3000, 64
    places = sorted({0, 1, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 1023, 1024, 2047, 2048, 2975, 2976, n - 2, n - 1})
    banner(f"paged attention {kind}: {len(places)} places of {n}")
    c = Cache(kind, 1, -(-n // 8) + 3, 8, 1, hd, False, 1).fill([n], rng, lambda r, s: grid(r, s) * 0)
    c.set_values(1, 0, 0, np.arange(n), grid(rng, (n, 1, hd)))
    for at in places:
        k = np.zeros((n, 1, hd), np.float32)
        k[at, 0, 5] = 2.0
        c.set_values(0, 0, 0, np.arange(n), k)
        c.upload()
        q = np.zeros((1, 2, hd), np.float32)
        q[0, :, 5] = 20.0
        got = c.run_attend(0, q, [0], 1.0)
        v = c.values(1, 0, 0, [at])[0, 0]
        assert np.abs(got - v).max() < 1e-5, at   # (the others weigh n e^-40)


def test_equals_the_contiguous_twin(lib):
    """A contiguous cache is a paged one with its pages in order."""
    banner("paged attention over the contiguous cache")
    rng = np.random.default_rng(11)
    n, ms, heads, kv, hd = 777, 1024, 16, 4, 128
    c = Cache("f16", 2, ms // 16, 16, kv, hd, False, 1)
    c.k[:], c.v[:] = encode(normal(rng, c.k.shape), "f16"), encode(normal(rng, c.v.shape), "f16")
    c.tables[0], c.lens[0] = np.arange(ms // 16), n
    c.upload()
    q = normal(rng, (1, heads, hd))
    got = c.run_attend(1, q, [0], 0.088)
    dq, out = D(q), D(np.zeros_like(q))
    lib.gsdh_gqa_attention(None, p(dq), p(c.dev["k"]), p(c.dev["v"]), p(out), 1, n - 1, heads, kv, hd, ms, 0.088)
    want = H(out, np.float32, q.size).reshape(q.shape)
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 1e-5


@pytest.mark.parametrize("scale_q", [1e-30, 1e-3, 1e4, 3e8])
def test_sizes_of_q(lib, scale_q):
    """q far from one: its parts are taken from a scaled copy (scores beyond 1e4 pick one position)."""
    rng = np.random.default_rng(5)
    c = Cache("f16", 1, 20, 16, 2, 128, False, 1).fill([300], rng, grid)
    q = (grid(rng, (1, 4, 128)) * scale_q).astype(np.float32)
    got = c.run_attend(0, q, [0], 1.0 / scale_q if scale_q < 1 else 0.05 / scale_q)
    check(got, *c.attend(0, q, [0], np.float32(1.0 / scale_q if scale_q < 1 else 0.05 / scale_q)), [300])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-42])
def test_scales(lib, scale):
    """No scale, a negative one, one below the normal range; negative and zero scales of an 8-bit cache."""
    rng = np.random.default_rng(15)
    for scales in (None, np.array([[[-0.5, 0.0]], [[-2.0, 0.25]]], np.float32)):
        c = Cache("e4m3", 1, 60, 8, 2, 64, False, 4, scales=np.ones((2, 1, 2), np.float32)).fill([0, 1, 50, 333], rng, grid)
        if scales is not None:
            c.scales = scales
            c.upload()
        q = grid(rng, (4, 8, 64))
        got = c.run_attend(0, q, range(4), scale)
        check(got, *c.attend(0, q, range(4), np.float32(scale)), [0, 1, 50, 333])


def test_infinities_and_nan(lib):
    """A NaN or an infinity among a sequence's own rows shows in its row alone
    (as an infinity or a NaN: the parts of P may differ in sign)."""
    banner("paged attention: NaN and infinities")
    rng = np.random.default_rng(6)
    c = Cache("f16", 1, 40, 16, 2, 64, False, 5).fill([100, 100, 100, 100, 100], rng, grid)
    nan, inf = np.uint16(0x7E00), np.uint16(0x7C00)
    c.k[c.rows(None, 0, [50], c.tables[1])] = nan
    c.v[c.rows(None, 0, [99], c.tables[2])] = nan
    at = c.rows(None, 0, [7], c.tables[3])
    c.v[at] = inf
    c.upload()
    q = grid(rng, (5, 4, 64))
    got = c.run_attend(0, q, range(5), 0.1)
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
    assert not np.isfinite(got[3]).any()
    want = c.attend(0, q[[0, 4]], [0, 4], np.float32(0.1))
    check(got[[0, 4]], *want, [100, 100], exact_dots=True)


def test_bad_pages_lengths_and_sequences(lib):
    """What lies outside the cache is not read: the row is NaN, the status word says so."""
    from gsdlq import hip
    banner("paged attention: tables, lengths and sequences outside the cache")
    rng = np.random.default_rng(7)
    c = Cache("f16", 1, 40, 16, 2, 64, False, 6, 8).fill([100, 100, 100, 100, 20, 0], rng, grid)
    c.tables[1, 3], c.tables[2, 6] = 40, -7
    c.lens[3], c.lens[5] = 8 * 16 + 1, -1
    c.upload()
    q = grid(rng, (8, 4, 64))
    seqs = [0, 1, 2, 3, 4, 5, 6, -1]
    got = c.run_attend(0, q, seqs, 0.1)
    for i in (1, 2, 3, 5, 6):
        assert np.isnan(got[i]).all(), i
    assert (got[7] == 7.0).all()
    c.lens[3] = c.lens[5] = 0
    want = c.attend(0, q[[0, 4]], [0, 4], np.float32(0.1))
    check(got[[0, 4]], *want, [100, 20], exact_dots=True)
    assert c.status() == hip.PAGES_BAD_INDEX


def test_workspace_serves_other_sizes(lib):
    """One workspace for calls of more and fewer rows and of other lengths;
    nothing behind it is written."""
    banner("paged attention: one workspace, many sizes")
    rng = np.random.default_rng(8)
    lens = list(rng.integers(0, 700, 40)) + [5000, 4000]
    c = Cache("f16", 1, sum(-(-int(n) // 32) for n in lens), 32, 4, 64, False, 42, 160).fill([int(n) for n in lens], rng, grid)
    need = lib.gsdh_paged_attention_workspace_bytes(c.at, 42, 16)
    ws = D(np.concatenate([np.zeros(need, np.uint8), np.full(4096, 0xA5, np.uint8)]))
    ws.nbytes = need
    q = grid(rng, (42, 16, 64))
    want = c.attend(0, q, range(42), np.float32(0.1))
    for rows in (range(42), [41], range(42), [40, 41, 3], range(35, 42), range(42)):
        rows = list(rows)
        got = c.run_attend(0, q[rows], rows, 0.1, ws=ws)
        check(got, *(w[rows] for w in want), [c.lens[r] for r in rows], exact_dots=True)
    ws.nbytes = need + 4096
    assert (H(ws, np.uint8)[need:need + 4096] == 0xA5).all()


def test_captured_and_replayed(lib):
    """One captured launch: q, lengths and tables as they are at each replay,
    eager calls on another workspace between the replays."""
    banner("paged attention: a captured launch")
    rng = np.random.default_rng(9)
    c = Cache("f16", 1, 400, 16, 2, 128, False, 3, 200).fill([3000, 17, 900], rng, grid)
    n, heads, hd = 3, 8, 128
    dq, ds = D(np.zeros((n, heads, hd), np.float32)), ints(range(3))
    out, ws, other = D(np.zeros((n, heads, hd), np.float32)), c.space(3, heads), c.space(3, heads)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(stream))

    def put(buf, a):
        a = np.ascontiguousarray(a)
        lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
        lib.gsdh_stream_sync(None)

    lib.gsdh_stream_begin_capture(stream)
    lib.gsdh_paged_attention(stream, c.at, 0, p(dq), heads * hd, p(ds), n, heads, 0.1, 0, p(out), heads * hd, p(ws), ws.nbytes)
    lib.gsdh_stream_end_capture(stream, ctypes.byref(graph))
    for lens in ([3000, 17, 900], [1, 0, 33], [2999, 17, 2], [128, 5, 900]):
        c.lens[:] = lens
        put(c.dev["lens"], c.lens)
        q = grid(rng, (n, heads, hd))
        put(dq, q)
        lib.gsdh_graph_replay(graph, stream)
        lib.gsdh_stream_sync(stream)
        got = H(out, np.float32, q.size).reshape(q.shape)
        check(got, *c.attend(0, q, range(3), np.float32(0.1)), lens, exact_dots=True)
        assert np.array_equal(got, c.run_attend(0, q, range(3), 0.1, ws=other))
    lib.gsdh_graph_destroy(graph)
    lib.gsdh_stream_destroy(stream)


def test_two_streams(lib):
    """Two launches in flight, each on its own stream and workspace."""
    banner("paged attention: two streams")
    rng = np.random.default_rng(10)
    c = Cache("e4m3", 1, 800, 16, 2, 128, False, 2, 400).fill([6000, 5000], rng, grid)
    heads, hd, streams, sets = 8, 128, [], []
    for s in range(2):
        h = ctypes.c_void_p()
        lib.gsdh_stream_create(ctypes.byref(h))
        streams.append(h)
        q = grid(rng, (1, heads, hd))
        sets.append((q, D(q), ints([s]), D(np.zeros_like(q)), c.space(1, heads)))
    for _ in range(20):
        for h, (q, dq, ds, out, ws) in zip(streams, sets):
            lib.gsdh_paged_attention(h, c.at, 0, p(dq), heads * hd, p(ds), 1, heads, 0.1, 0, p(out), heads * hd, p(ws), ws.nbytes)
    for s, (h, (q, dq, ds, out, ws)) in enumerate(zip(streams, sets)):
        lib.gsdh_stream_sync(h)
        got = H(out, np.float32, q.size).reshape(q.shape)
        check(got, *c.attend(0, q, [s], np.float32(0.1)), [c.lens[s]], exact_dots=True)
    for h in streams:
        lib.gsdh_stream_destroy(h)


def test_many_rows(lib):
    """More rows than a wave has lanes, several per lane, on shared pages."""
    banner("paged attention: 1500 rows")
    rng = np.random.default_rng(12)
    lens = [int(n) for n in rng.integers(0, 90, 60)]
    c = Cache("f16", 1, 400, 16, 1, 64, False, 60, 8).fill(lens, rng, grid)
    seqs = rng.integers(-1, 60, 1500)
    q = grid(rng, (1500, 2, 64))
    got = c.run_attend(0, q, seqs, 0.1)
    want = c.attend(0, q, seqs, np.float32(0.1))
    check(got, *want, [c.lens[s] if s >= 0 else 0 for s in seqs], exact_dots=True)
    assert (got[seqs < 0] == 7.0).all()


def test_pool_beyond_4_gib(lib):
    """Pages whose offset passes 2^32 bytes, in the second layer of a large pool."""
    banner("paged attention: a 5 GiB pool")
    rng = np.random.default_rng(13)
    page, kv, hd, pages, n = 256, 8, 128, 5000, 700   # 512 KiB a page
    bytes_ = 2 * pages * page * kv * hd * 2
    bufs = []
    for _ in range(2):
        b = ctypes.c_void_p()
        lib.gsdh_malloc(ctypes.byref(b), bytes_)
        bufs.append(b)
    small = Cache("f16", 1, 3, page, kv, hd, False, 1, 4).fill([n], rng, grid)
    far = [pages - 1, 17, pages - 2]
    tables = np.full((1, 4), -1, np.int32)
    tables[0, :3] = far
    for buf, pool in zip(bufs, (small.k, small.v)):
        for j, pg in enumerate(far):
            src = np.ascontiguousarray(pool[0, small.tables[0, j]])
            at = (pages + pg) * page * kv * hd * 2
            lib.gsdh_memcpy_h2d(ctypes.c_void_p(buf.value + at), src.ctypes.data_as(ctypes.c_void_p), src.nbytes, None)
            lib.gsdh_stream_sync(None)
    dt = D(tables)
    c = small.struct(k=bufs[0], v=bufs[1], n_layers=2, n_pages=pages, tables=dt.ptr, refs=None)
    q = grid(rng, (1, 16, hd))
    dq, out, ds = D(q), D(np.zeros_like(q)), ints([0])
    ws = small.space(1, 16)
    lib.gsdh_paged_attention(None, ctypes.byref(c), 1, p(dq), 16 * hd, p(ds), 1, 16, 0.1, 0, p(out), 16 * hd, p(ws), ws.nbytes)
    got = H(out, np.float32, q.size).reshape(q.shape)
    check(got, *small.attend(0, q, [0], np.float32(0.1)), [n], exact_dots=True)
    for b in bufs:
        lib.gsdh_free(b)
