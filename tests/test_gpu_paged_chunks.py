"""gsdh_paged_chunk_attention against softmax(q K) V in 64 bits over what each
row sees.

Tolerances, per output element, in units of sum P |V|: a score is off by at most
(hd + 16) half steps of fp32 of scale * sum |q k| (its accumulation, the split of
q; nothing where the products are exact) and 8 of |s| (scaling, exponential), so
P by twice that; the sum of the weights adds every second position in one lane
(n / 2 roundings), the outputs 16 positions at a time (n / 16, and n / 64 for
the running maximum), the join and the rest less than 160.  Beside that, each
weight may lose 2^-38 of the largest one (chunk_util.check).  Rows of 16 bits: half
a step of each weight and of the output."""
import numpy as np
import pytest

from chunk_util import attend_chunks, check, chunk_cache, rounded, run_chunks, space
from gpu_util import D, H, banner, p
from paged_util import encode, grid, ints, nan_bits, normal

pytestmark = pytest.mark.gpu
TYPES = [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("e4m3", "f32"), ("e4m3", "f16"), ("e4m3", "bf16")]


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


LENS = [0, 1, 2, 9, 40, 63, 64, 65, 130, 200, 300]
NEW = [0, 1, 2, 3, 40, 1, 17, 64, 130, 5, 0]


def ragged(order=(10, 4, 8, 0, 9, 7, 6, 5, 3, 2, 1)):
    """Chunks in that order, with padding of 2 rows behind the third, one row that nobody names at the end."""
    seqs, starts = [], [0]
    for n, s in enumerate(order):
        seqs.append(s)
        starts.append(starts[-1] + NEW[s])
        if n == 2:
            seqs.append(-1)
            starts.append(starts[-1] + 2)
    return seqs, starts


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
@pytest.mark.parametrize("heads,kv,hd,page,head_major", [(4, 2, 64, 8, False), (8, 2, 128, 16, True), (4, 4, 128, 128, False), (6, 2, 64, 32, True),
                                                         (16, 2, 256, 8, True), (16, 1, 128, 16, False), (1, 1, 64, 256, False), (7, 1, 128, 8, False)])
def test_ragged_batch(lib, kind, rows, heads, kv, hd, page, head_major, few_rows):
    """Every length and chunk, padding, NaN wherever nobody wrote, padded strides."""
    banner(f"chunks {kind} {rows} {heads}/{kv}x{hd} page {page} {'head' if head_major else 'slot'}")
    rng = np.random.default_rng(heads * hd + page)
    c = chunk_cache(kind, LENS, page, kv, hd, head_major, rng, grid, layers=2, few_rows=few_rows)
    seqs, starts = ragged()
    q, scale = grid(rng, (starts[-1] + 1, heads, hd)), 1.0 / float(np.sqrt(hd))
    got = run_chunks(c, 1, q, rows, seqs, starts, scale, q_pad=8, out_pad=16)
    check(got, attend_chunks(c, 1, q, seqs, starts, scale), rows, exact_dots=True)
    assert c.status() == 0


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
@pytest.mark.parametrize("window", [1, 7, 64, 65, 150, 100000])
def test_window(lib, kind, rows, window, few_rows):
    banner(f"chunks {kind} {rows} window {window}")
    rng = np.random.default_rng(window)
    c = chunk_cache(kind, LENS, 16, 2, 64, False, rng, grid, few_rows=few_rows)
    for s, n in enumerate(LENS):   # what the window leaves behind may hold anything
        gone = np.arange(max(0, n - NEW[s] + 1 - window))
        if len(gone):
            for pool in (c.k, c.v):
                pool[c.rows(None, 0, gone, c.tables[s])] = nan_bits((len(gone), 2, 64), kind)
    c.upload()
    seqs, starts = ragged()
    q, scale = grid(rng, (starts[-1] + 1, 6, 64)), 0.11
    got = run_chunks(c, 0, q, rows, seqs, starts, scale, window)
    check(got, attend_chunks(c, 0, q, seqs, starts, np.float32(scale), window), rows, exact_dots=True)


@pytest.mark.parametrize("kind,rows,heads,kv,hd,lens,new", [
    ("f16", "f32", 32, 8, 128, [8192, 3000, 77], [5, 1, 33]), ("bf16", "f32", 8, 2, 128, [20011, 5], [3, 5]),
    ("e4m3", "f32", 16, 2, 64, [12345, 999], [2, 40]), ("f16", "f16", 4, 1, 256, [9001], [7]), ("bf16", "bf16", 4, 1, 128, [30001, 64], [4, 1]),
    ("e4m3", "bf16", 8, 8, 128, [5000], [1])])
def test_long_split_and_joined(lib, kind, rows, heads, kv, hd, lens, new):
    """Few rows over long contexts, any values: split over many blocks and joined, the same bits twice."""
    banner(f"chunks {kind} {rows} {heads}/{kv}x{hd} over {lens}")
    rng = np.random.default_rng(lens[0])
    c = chunk_cache(kind, lens, 64, kv, hd, True, rng, normal)
    starts = np.cumsum([0] + new).tolist()
    q, scale = rounded(1.5 * normal(rng, (starts[-1], heads, hd)), rows).astype(np.float32), 1.0 / float(np.sqrt(hd))
    ws = space(c, len(lens), starts[-1], heads)
    got = run_chunks(c, 0, q, rows, None, starts, scale, ws=ws)
    check(got, attend_chunks(c, 0, q, None, starts, np.float32(scale)), rows)
    for _ in range(3):
        assert np.array_equal(got, run_chunks(c, 0, q, rows, None, starts, scale, ws=ws, repeat=2))


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt(lib, kind, rows, hd, few_rows):
    """A prompt from its first token on, and the same in two pieces."""
    banner(f"prompt {kind} {rows} hd {hd}")
    rng = np.random.default_rng(hd)
    m, heads, kv = 401, 4, 2
    c = chunk_cache(kind, [m], 16, kv, hd, False, rng, normal, few_rows=few_rows)
    q, scale = rounded(normal(rng, (m, heads, hd)), rows).astype(np.float32), 1.0 / float(np.sqrt(hd))
    want = attend_chunks(c, 0, q, [0], [0, m], np.float32(scale))
    got = run_chunks(c, 0, q, rows, [0], [0, m], scale)
    check(got, want, rows)
    c.lens[0] = 150
    c.upload()
    first = run_chunks(c, 0, q[:150], rows, [0], [0, 150], scale)
    c.lens[0] = m
    c.upload()
    rest = run_chunks(c, 0, q[150:], rows, [0], [0, m - 150], scale)
    check(np.concatenate([first, rest]), want, rows)


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
def test_one_token_is_decode(lib, kind, hd, few_rows):
    """Chunks of one token against the decode attention, over the same cache and rows."""
    banner(f"one token {kind} hd {hd}")
    rng = np.random.default_rng(5)
    lens = [1, 63, 64, 65, 700]
    c = chunk_cache(kind, lens, 16, 2, hd, False, rng, normal, few_rows=few_rows)
    q, starts, seqs = normal(rng, (5, 8, hd)), list(range(6)), [4, 2, 0, 1, 3]
    got = run_chunks(c, 0, q, "f32", seqs, starts, 0.125)
    want = attend_chunks(c, 0, q, seqs, starts, 0.125)
    check(got, want, "f32")
    check(c.run_attend(0, q, seqs, 0.125).astype(np.float64), want, "f32")


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
def test_every_position_counts(lib, kind, rows, few_rows):
    """One position that outweighs all others: the rows from it on give its V row, those before it none of it."""
    rng = np.random.default_rng(3)
    n, m, hd = 1000, 200, 64
    places = [0, 1, 31, 32, 63, 64, 127, 500, 799, 800, 801, 831, 832, 863, 895, 896, 998, 999]
    banner(f"chunks {kind} {rows}: {len(places)} places of {n}")
    c = chunk_cache(kind, [n], 8, 1, hd, False, rng, lambda r, s: grid(r, s) * 0, few_rows=few_rows)
    c.set_values(1, 0, 0, np.arange(n), grid(rng, (n, 1, hd)))
    q = np.zeros((m, 2, hd), np.float32)
    q[:, :, 5] = 20.0
    for at in places:
        k = np.zeros((n, 1, hd), np.float32)
        k[at, 0, 5] = 2.0
        c.set_values(0, 0, 0, np.arange(n), k)
        c.upload()
        got = run_chunks(c, 0, q, rows, [0], [0, m], 1.0)
        check(got, attend_chunks(c, 0, q, [0], [0, m], 1.0), rows, exact_dots=True)


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 70])
def test_what_a_row_does_not_see(lib, kind, rows, bad, window, few_rows):
    """A NaN or an infinity in V or K: rows that do not see it are as without it, those that do are not finite in
    that dim (V) or of that KV head (K)."""
    if kind == "e4m3" and not np.isnan(bad):
        pytest.skip("e4m3 has no infinities")
    banner(f"unseen {kind} {rows} {bad} window {window}")
    rng = np.random.default_rng(11)
    n, m, kv, heads, hd, at, dim = 300, 150, 2, 4, 64, 230, 37
    c = chunk_cache(kind, [n], 16, kv, hd, False, rng, grid, few_rows=few_rows)
    q = grid(rng, (m, heads, hd))
    want = attend_chunks(c, 0, q, [0], [0, m], 0.1, window)
    clean = run_chunks(c, 0, q, rows, [0], [0, m], 0.1, window)
    check(clean, want, rows, exact_dots=True)
    pos = n - m + np.arange(m)
    sees = (pos >= at) & ((pos - at < window) if window else True)
    for pool in (c.v, c.k):
        keep = pool.copy()
        idx = c.rows(None, 0, np.array([at]), c.tables[0])
        row = pool[idx].copy()
        row[0, 1, dim] = encode(np.float32(bad), kind)
        pool[idx] = row
        c.upload()
        got = run_chunks(c, 0, q, rows, [0], [0, m], 0.1, window)
        assert np.array_equal(got[~sees], clean[~sees])
        assert np.array_equal(got[:, :2], clean[:, :2])     # the other KV head
        if pool is c.v:
            assert not np.isfinite(got[sees][:, 2:, dim]).any()
            others = np.arange(hd) != dim
            assert np.array_equal(got[:, :, others], clean[:, :, others])
        elif np.isnan(bad):
            assert np.isnan(got[sees][:, 2:]).all()
        pool[...] = keep
    c.upload()


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", TYPES)
def test_no_weight_at_all(lib, kind, rows, few_rows):
    """Scores that are all -inf are NaN, one that is not takes all; NaN in q stays with its row and head."""
    if kind == "e4m3":
        pytest.skip("e4m3 has no infinities")
    rng = np.random.default_rng(2)
    n, m, hd = 100, 100, 64
    c = chunk_cache(kind, [n], 16, 1, hd, False, rng, grid, few_rows=few_rows)
    k = np.zeros((n, 1, hd), np.float32)
    k[:50, 0, 3] = -np.inf
    c.set_values(0, 0, 0, np.arange(n), k)
    c.upload()
    q = np.zeros((m, 2, hd), np.float32)
    q[:, :, 3] = 2 + 2.0 ** -8 + 2.0 ** -12 + 2.0 ** -16   # (above 0 in every 16-bit part)
    q[60, 1, 7] = np.nan
    got = run_chunks(c, 0, q, rows, [0], [0, m], 0.5)
    assert np.isnan(got[:50]).all() and np.isnan(got[60, 1]).all()
    v = c.values(1, 0, 0, np.arange(n))[:, 0]
    ok = [t for t in range(50, n) if t != 60]
    want = np.stack([v[50:t + 1].mean(0) for t in ok])
    tol = 2.0 ** (-10 if rows == "f16" else -7 if rows == "bf16" else -20) * np.abs(v).max()
    assert np.abs(got[ok] - want[:, None]).max() <= tol


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("n,m", [(200, 70), (6000, 3)])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_the_ends_of_bf16(lib, rows, n, m, few_rows):
    """Finite rows over all of the type's range give finite results; scores far beyond fp32 after scaling keep the
    largest weight at 1, within a block and over many; a scale of 0 weighs all alike."""
    rng, hd = np.random.default_rng(4), 64
    huge = 2.0 ** 127
    c = chunk_cache("bf16", [n], 16, 1, hd, False, rng, grid, few_rows=few_rows)
    v = np.sign(grid(rng, (n, 1, hd)) + 0.1) * huge
    c.set_values(1, 0, 0, np.arange(n), v)
    k = grid(rng, (n, 1, hd)) * np.float32(2.0 ** 120)
    c.set_values(0, 0, 0, np.arange(n), k)
    c.upload()
    q = grid(rng, (m, 2, hd)) * np.float32(2.0 ** 120)
    for scale in (0.125, -0.125, 0.0):
        got = run_chunks(c, 0, q, rows, [0], [0, m], scale)
        assert np.isfinite(got).all()
        pos = n - m + np.arange(m)
        kk, vv = c.values(0, 0, 0, np.arange(n))[:, 0] / 2.0 ** 120, c.values(1, 0, 0, np.arange(n))[:, 0]
        for t in sorted({0, 1, min(33, m - 1), m - 1}):
            x = kk[:pos[t] + 1] @ (q[t, 0].astype(np.float64) / 2.0 ** 120)
            if scale == 0:
                want = vv[:pos[t] + 1].mean(0)
            else:
                x = x * np.sign(scale)
                want = vv[:pos[t] + 1][x == x.max()].mean(0)
            tol = (2.0 ** -16 if rows == "f32" else 2.0 ** -7) * huge
            assert np.abs(got[t, 0] - want).max() <= tol, (scale, t)


@pytest.mark.parametrize("few_rows", [False, True])
def test_scales(lib, few_rows):
    """Negative, zero and large scales over fp16, fp32 and fp16 rows; one of NaN makes NaN."""
    rng = np.random.default_rng(8)
    c = chunk_cache("f16", [150], 16, 2, 64, False, rng, grid, few_rows=few_rows)
    q = grid(rng, (60, 4, 64))
    for rows in ("f32", "f16"):
        for scale in (-0.3, 0.0, -0.0, 40.0, 1e-30):
            got = run_chunks(c, 0, q, rows, [0], [0, 60], scale)
            check(got, attend_chunks(c, 0, q, [0], [0, 60], float(np.float32(scale))), rows, exact_dots=True)
        assert np.isnan(run_chunks(c, 0, q, rows, [0], [0, 60], np.nan)).all()


@pytest.mark.parametrize("few_rows", [False, True])
def test_bad_indices(lib, few_rows):
    """Left out or NaN, reported, and nothing else touched."""
    from gsdlq import hip
    rng = np.random.default_rng(1)
    lens = [100, 50, 40, 30, 200, 64]
    c = chunk_cache("f16", lens, 16, 2, 64, False, rng, grid, few_rows=few_rows)
    q = grid(rng, (60, 4, 64))

    def run(seqs, starts, **kw):
        c.clear_status()
        return run_chunks(c, 0, q, "f32", seqs, starts, 0.2, **kw)

    want = lambda seqs, starts: attend_chunks(c, 0, q, seqs, starts, np.float32(0.2))[0]  # noqa: E731
    good = want([0, 5], [0, 10, 30])
    # a sequence outside the cache, beside good ones
    got = run([0, 6, 5], [0, 10, 12, 32])
    assert c.status() == hip.PAGES_BAD_INDEX and np.isnan(got[10:12]).all() and (got[32:] == 7).all()
    assert np.abs(got[:10] - good[:10]).max() < 1e-5 and np.isfinite(got[12:32]).all()
    # a chunk longer than its sequence
    got = run([3, 0], [0, 31, 41])
    assert c.status() == hip.PAGES_BAD_INDEX and np.isnan(got[:31]).all() and np.isfinite(got[31:41]).all()
    # starts that fall or lie outside
    for starts in ([10, 5, 20], [-3, 0, 20], [0, 61, 61], [0, 100, 120]):
        got = run([0, 5], starts)
        assert c.status() == hip.PAGES_BAD_INDEX
        for i in range(2):
            a, b = starts[i], starts[i + 1]
            if 0 <= a <= b <= 60 and b > a:
                assert np.isfinite(got[a:b]).all()
        assert (got[20:] == 7).all()
    # a length beyond the table
    keep = c.lens.copy()
    c.lens[0] = c.width * c.page + 1
    c.upload()
    got = run([0, 5], [0, 10, 30])
    assert c.status() == hip.PAGES_BAD_INDEX and np.isnan(got[:10]).all() and np.isfinite(got[10:30]).all()
    c.lens[:] = keep
    # a page outside the pool: rows that see it
    for page in (-1, c.pages, 1 << 30):
        old = c.tables[0, 5]
        c.tables[0, 5] = page    # positions 80 .. 95
        c.upload()
        got = run([0, 5], [0, 40, 60])
        assert c.status() == hip.PAGES_BAD_INDEX
        assert np.isfinite(got[:20]).all() and np.isnan(got[20:40]).all() and np.isfinite(got[40:60]).all()
        c.clear_status()
        got = run_chunks(c, 0, q, "f16", [0, 5], [0, 40, 60], 0.2, window=3)
        assert np.isfinite(got[:20]).all() and np.isnan(got[20:38]).all() and np.isfinite(got[38:60]).all()
        c.tables[0, 5] = old
    c.upload()


def test_one_row_of_q_for_all(lib):
    """A stride of 0: every token has the same q."""
    rng = np.random.default_rng(6)
    c = chunk_cache("f16", [90], 16, 1, 64, False, rng, grid)
    q = np.repeat(grid(rng, (1, 2, 64)), 30, 0)
    dq, out, dt, ws = D(q[0]), D(np.full((30, 128), 7.0, np.float32)), ints([0, 30]), space(c, 1, 30, 2)
    lib.gsdh_paged_chunk_attention(None, c.at, 0, p(dq), 0, 0, None, p(dt), 1, 30, 2, 0.2, 0, p(out), 128, p(ws), ws.nbytes)
    check(H(out, np.float32, 30 * 128).reshape(30, 2, 64).astype(np.float64), attend_chunks(c, 0, q, [0], [0, 30], np.float32(0.2)), "f32", True)


@pytest.mark.parametrize("few_rows", [False, True])
def test_replayed_while_sequences_grow(lib, few_rows):
    """A captured call reads lengths, starts and lists when it runs; every replay against the definition, eager work between."""
    import ctypes
    rng = np.random.default_rng(9)
    lens = [500, 40, 300]
    c = chunk_cache("f16", lens, 16, 2, 64, False, rng, grid, few_rows=few_rows)
    tokens, heads = 50, 4
    q = grid(rng, (tokens, heads, 64))
    dq, out, ws = D(q), D(np.zeros((tokens, heads * 64), np.float32)), space(c, 3, tokens, heads)
    dt, ds = ints([0, 0, 0, 0]), ints([0, 1, 2])
    st, ge = ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(st))
    lib.gsdh_stream_begin_capture(st)
    lib.gsdh_paged_chunk_attention(st, c.at, 0, p(dq), 0, heads * 64, p(ds), p(dt), 3, tokens, heads, 0.2, 0, p(out), heads * 64, p(ws), ws.nbytes)
    lib.gsdh_stream_end_capture(st, ctypes.byref(ge))

    def put(buf, a):
        a = np.ascontiguousarray(a)
        lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
        lib.gsdh_stream_sync(None)

    for now, seqs, starts in (([500, 40, 300], [0, 1, 2], [0, 5, 45, 50]), ([77, 3, 299], [2, 0, -1], [0, 50, 50, 50]),
                              ([500, 0, 1], [1, 2, 0], [0, 0, 1, 30]), ([500, 40, 300], [0, 1, 2], [0, 5, 45, 50])):
        c.lens[:] = now
        put(c.dev["lens"], c.lens)
        put(ds, np.asarray(seqs, np.int32))
        put(dt, np.asarray(starts, np.int32))
        put(out, np.full((tokens, heads * 64), 7.0, np.float32))
        lib.gsdh_graph_replay(ge, st)
        lib.gsdh_stream_sync(st)
        got = H(out, np.float32, tokens * heads * 64).reshape(tokens, heads, 64).astype(np.float64)
        check(got, attend_chunks(c, 0, q, seqs, starts, np.float32(0.2)), "f32", True)
        eager = run_chunks(c, 0, q, "f32", seqs, starts, 0.2)
        assert np.array_equal(got, eager)
    assert c.status() == 0
    lib.gsdh_graph_destroy(ge)
    lib.gsdh_stream_destroy(st)


def test_two_streams(lib):
    """Two calls at once, a workspace each."""
    import ctypes
    rng = np.random.default_rng(10)
    c = chunk_cache("bf16", [4000, 900], 16, 2, 64, False, rng, normal)
    q = normal(rng, (40, 4, 64))
    want = attend_chunks(c, 0, q, [0, 1], [0, 20, 40], np.float32(0.125))
    dq, dt, sts, outs, spaces = D(q), ints([0, 20, 40]), [], [], []
    for _ in range(2):
        st = ctypes.c_void_p()
        lib.gsdh_stream_create(ctypes.byref(st))
        sts.append(st)
        outs.append(D(np.full((40, 256), 7.0, np.float32)))
        spaces.append(space(c, 2, 40, 4))
    for _ in range(10):
        for st, out, ws in zip(sts, outs, spaces):
            lib.gsdh_paged_chunk_attention(st, c.at, 0, p(dq), 0, 256, None, p(dt), 2, 40, 4, 0.125, 0, p(out), 256, p(ws), ws.nbytes)
    for st, out in zip(sts, outs):
        lib.gsdh_stream_sync(st)
        check(H(out, np.float32, 40 * 256).reshape(40, 4, 64).astype(np.float64), want, "f32")
        lib.gsdh_stream_destroy(st)


@pytest.mark.parametrize("few_rows", [False, True])
def test_many_chunks(lib, few_rows):
    """More chunks than a wave has lanes, most of them of one token."""
    banner("200 chunks")
    rng = np.random.default_rng(12)
    lens = [1 + (37 * i) % 90 for i in range(200)]
    c = chunk_cache("f16", lens, 8, 1, 64, False, rng, grid, few_rows=few_rows)
    new = [1 if i % 9 else min(n, 30) for i, n in enumerate(lens)]
    starts = np.cumsum([0] + new).tolist()
    q = grid(rng, (starts[-1], 2, 64))
    got = run_chunks(c, 0, q, "f32", None, starts, 0.2)
    check(got, attend_chunks(c, 0, q, None, starts, np.float32(0.2)), "f32", True)
