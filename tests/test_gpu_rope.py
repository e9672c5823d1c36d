"""gsdh_rope_rows and gsdh_paged_rope_append against the rotation in 64 bits.

Tolerances: the angle's turns are exact to 2^-30 (positions below 2^24) and their
fraction, at most half a turn, is rounded once to fp32 (2^-26 of a turn, 2^-23.3
radians); cosine and sine are within 2 units of 2^-24 and multiplied by the scale (half
a step), the products and the sum add three half steps.  Each of the two terms is so
off by less than 2^-23.3 + 2 * 2^-24 + 4 * 2^-24 < 2^-20.9 of |scale| (|u| + |v|); then
half a step of the row's or the cache's type."""
import ctypes

import numpy as np
import pytest

from chunk_util import HALF, row_bits, row_values, rounded
from gpu_util import D, H, banner, p
from paged_util import Cache, decode, encode, grid, ints, nan_bits, normal

pytestmark = pytest.mark.gpu
TURN = 2.0 ** -20.9
LEAST = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0, "e4m3": 2.0 ** -10}   # half of the least number, where rows reach it
KV_HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()
    return hip.lib()


def frequencies(lib, rd, kind="plain", factor=1.0):
    from gsdlq import hip
    f = np.empty(rd // 2)
    lib.gsdh_rope_frequencies(hip.ROPE_KINDS[kind], 1e6, rd, factor, 8192.0, 1.0, 4.0, hip.ptr(f))
    return f


def rope(freqs, interleaved, scale=1.0):
    """(device buffer that the struct names, struct)"""
    from gsdlq import hip
    d = D(freqs)
    return d, hip.GsdRope(freqs=d.ptr, rotary_dim=2 * len(freqs), interleaved=interleaved, scale=scale)


def turn(x, freqs, pos, interleaved, scale=1.0):
    """float64 (rows, what their error is in units of TURN); x [n, heads, hd]."""
    x = np.asarray(x, np.float64)
    a = np.asarray(pos, np.float64)[:, None, None] * freqs
    c, s = np.cos(a) * scale, np.sin(a) * scale
    y, mag, r = x.copy(), np.zeros_like(x), 2 * len(freqs)
    i, j = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
    u, v = x[..., i], x[..., j]
    y[..., i], y[..., j] = u * c - v * s, u * s + v * c
    mag[..., i] = mag[..., j] = abs(scale) * (np.abs(u) + np.abs(v))
    return y, mag


def run_rows(lib, q, rows, freqs, pos, interleaved, scale=1.0, in_place=False, pad=0, out_pad=0):
    from gsdlq import hip
    n, heads, hd = q.shape
    w = heads * hd
    src = np.full((n, w + pad), 3.0, np.float32)
    src[:, :w] = q.reshape(n, w)
    d, r = rope(freqs, interleaved, scale)
    dx, dp = D(row_bits(src, rows)), ints(pos)
    one = row_bits(np.float32(5), rows)
    do = dx if in_place else D(np.full((n, w + out_pad), one, one.dtype))
    stride = w + (pad if in_place else out_pad)
    lib.gsdh_rope_rows(None, ctypes.byref(r), p(dx), hip.ROW_TYPES[rows], w + pad, p(do), stride, p(dp), n, heads, hd)
    out = row_values(H(do, one.dtype, n * stride).reshape(n, stride), rows)
    assert (out[:, w:] == (3 if in_place else 5)).all()
    return out[:, :w].reshape(n, heads, hd)


def within(got, want, mag, half, least):
    off = np.abs(got - want) - (TURN * mag + half * (np.abs(want) + TURN * mag) + least)
    assert np.isfinite(got).all() and off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("heads,hd,rd", [(40, 128, 128), (1, 64, 16), (3, 96, 24), (5, 80, 20), (2, 8, 2), (7, 128, 50), (33, 64, 32), (1, 1024, 1024),
                                         (2, 256, 254)])
def test_rows(lib, rows, interleaved, heads, hd, rd):
    """Whole heads and parts of them, odd ones too, near and far positions, in place and not, padded strides."""
    banner(f"rope {rows} {heads}x{hd} of {rd} {'pairs' if interleaved else 'halves'}")
    rng = np.random.default_rng(hd + rd)
    pos = np.array([0, 1, 2, 77, 4095, 131071, 1000003, -1, -4095, 5, 5, 12345678])
    f = frequencies(lib, rd)
    q = rounded(normal(rng, (len(pos), heads, hd)), rows).astype(np.float32)
    for scale in (1.0, 1.25):
        want, mag = turn(q, f, pos, interleaved, scale)
        got = run_rows(lib, q, rows, f, pos, interleaved, scale, pad=8, out_pad=16)
        within(got, want, mag, HALF[rows], LEAST[rows])
        assert np.array_equal(got[..., rd:], q[..., rd:])
        assert np.array_equal(got, run_rows(lib, q, rows, f, pos, interleaved, scale, in_place=True, pad=8))


@pytest.mark.parametrize("kind", ["linear", "ntk", "by_parts"])
def test_scaled_contexts(lib, kind):
    rng = np.random.default_rng(1)
    f = frequencies(lib, 128, kind, 8.0)
    pos = rng.integers(0, 1 << 20, 50)
    q = normal(rng, (50, 4, 128))
    want, mag = turn(q, f, pos, 0)
    within(run_rows(lib, q, "f32", f, pos, 0), want, mag, HALF["f32"], 0)


def test_undone_and_gradient(lib):
    """Turning by -p undoes p; as the rows' gradient it agrees with differences of sum(g * y)."""
    rng = np.random.default_rng(2)
    f, pos = frequencies(lib, 32), rng.integers(0, 100000, 9)
    q, g = normal(rng, (9, 3, 64)), normal(rng, (9, 3, 64))
    y = run_rows(lib, q, "f32", f, pos, 1)
    back = run_rows(lib, y.astype(np.float32), "f32", f, -pos, 1)
    pair = np.maximum(np.abs(q[..., 0::2]), np.abs(q[..., 1::2])).repeat(2, -1)
    assert (np.abs(back - q) <= 6 * TURN * pair + 1e-30).all()
    grad = run_rows(lib, g, "f32", f, -pos, 1, 1.5)
    for t, h, d in ((0, 0, 0), (3, 1, 31), (8, 2, 7), (4, 0, 40)):
        step = np.zeros(q.shape)
        step[t, h, d] = 0.5
        diff = ((turn(q + step, f, pos, 1, 1.5)[0] - turn(q - step, f, pos, 1, 1.5)[0]) * g).sum()   # (linear: exact at any step)
        pair = np.abs(g[t, h, d // 2 * 2:d // 2 * 2 + 2]).sum()
        want = diff if d < 32 else g[t, h, d]
        assert abs(grad[t, h, d] - want) <= 1.5 * 2 * TURN * pair + 1e-12


def test_nan_and_infinities_stay_with_their_pairs(lib):
    rng = np.random.default_rng(3)
    f, pos = frequencies(lib, 20), np.array([3, 4])
    for interleaved in (0, 1):
        q = normal(rng, (2, 2, 64))
        clean = run_rows(lib, q, "f32", f, pos, interleaved)
        q[0, 1, 4], q[1, 0, 30] = np.inf, np.nan
        got = run_rows(lib, q, "f32", f, pos, interleaved)
        touched = np.zeros(q.shape, bool)
        touched[0, 1, [4, 5] if interleaved else [4, 14]] = True
        touched[1, 0, 30] = True
        assert not np.isfinite(got[touched]).any() and np.array_equal(got[~touched], clean[~touched])


def append(c, layer, rows, q, k, v, seqs, pos, freqs, interleaved, scale=1.0, in_place=False, stream=None):
    from gsdlq import hip
    n, heads, hd = q.shape
    fused = np.concatenate([x.reshape(n, -1) for x in (q, k, v)], 1)
    w, kw, es = heads * hd, c.kv * hd, 4 if rows == "f32" else 2
    d, r = rope(freqs, interleaved, scale)
    buf, ds, dp = D(row_bits(fused, rows)), ints(seqs), ints(pos)
    one = row_bits(np.float32(7), rows)
    out = buf if in_place else D(np.full((n, w), one, one.dtype))
    at = lambda i: ctypes.c_void_p(buf.ptr.value + es * i)  # noqa: E731
    st = w + 2 * kw
    c.lib.gsdh_paged_rope_append(stream, c.at, layer, ctypes.byref(r), hip.ROW_TYPES[rows], at(0), st, at(w), st, at(w + kw), st, p(out),
                                 st if in_place else w, p(ds), p(dp), n, heads)
    got = row_values(H(out, one.dtype, n * (st if in_place else w)).reshape(n, -1)[:, :w], rows)
    return got.reshape(n, heads, hd)


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,rd,interleaved,page,head_major", [
    (8, 2, 128, 128, 1, 16, False), (4, 4, 64, 16, 0, 8, True), (6, 2, 64, 20, 0, 32, False), (2, 1, 256, 64, 1, 128, True), (6, 3, 64, 50, 1, 8, False)])
def test_append(lib, kind, rows, heads, kv, hd, rd, interleaved, page, head_major):
    """Tokens of several sequences, padding and what is left out; nothing else in the pools changes."""
    from gsdlq import hip
    banner(f"append {rows} to {kind} {heads}/{kv}x{hd} of {rd}")
    rng = np.random.default_rng(hd + rd + page)
    lens = [70, 1, 33, 200]
    c = Cache(kind, 2, sum(-(-n // page) for n in lens) + 4, page, kv, hd, head_major, 5, 200 // page + 2).fill(lens + [0], rng, grid)
    c.refs[c.tables[3, 0]] = 2       # the first page of sequence 3 has two holders
    c.upload()
    seqs = [0, 0, 2, -1, 3, 3, 1, 4, 0, 0, 7, 2]
    pos = [69, 5, 32, 3, 199, 0, 0, 0, 70, -1, 0, 31]
    left = {3: 0, 5: hip.PAGES_SHARED, 7: hip.PAGES_BAD_INDEX, 8: hip.PAGES_BAD_INDEX, 9: hip.PAGES_BAD_INDEX, 10: hip.PAGES_BAD_INDEX}
    n = len(seqs)
    q, k, v = (rounded(2 * normal(rng, (n, h, hd)), rows).astype(np.float32) for h in (heads, kv, kv))
    f = frequencies(lib, rd, "by_parts", 4.0)
    want_q, mag_q = turn(q, f, pos, interleaved, 1.1)
    want_k, mag_k = turn(k, f, pos, interleaved, 1.1)
    before = c.download("k"), c.download("v")
    for in_place in (False, True):
        got = append(c, 1, rows, q, k, v, seqs, pos, f, interleaved, 1.1, in_place)
        ok = [t for t in range(n) if t not in left]
        within(got[ok], want_q[ok], mag_q[ok], HALF[rows], LEAST[rows])
        gone = sorted(left)
        assert np.array_equal(got[gone], q[gone] if in_place else np.full_like(got[gone], 7))
        assert c.status() == hip.PAGES_BAD_INDEX | hip.PAGES_SHARED
        written = np.zeros(before[0].shape, bool)
        for which, (pool, rows_, mag) in enumerate(((c.download("k"), want_k, mag_k), (c.download("v"), v.astype(np.float64), np.zeros(v.shape)))):
            written[...] = False
            for t in ok:
                at = c.rows(None, 1, np.array([pos[t]]), c.tables[seqs[t]])
                written[at] = True
                x = rows_[t] / (1 if c.scales is None else c.scales[which, 1].astype(np.float64)[:, None])
                m = mag[t] / (1 if c.scales is None else c.scales[which, 1].astype(np.float64)[:, None])
                limit = 448.0 if kind == "e4m3" else np.inf
                within(decode(pool[at], kind)[0], np.clip(x, -limit, limit), m + np.abs(x) * 2.0 ** -3, KV_HALF[kind], LEAST[kind])
            assert np.array_equal(pool[~written], before[which][~written])


def test_append_is_the_store_on_equal_angles(lib):
    """A whole head at positions whose angles fp32 holds exactly: the same K, V bits as the store with a table."""
    from paged_util import angles
    rng = np.random.default_rng(7)
    lens = [50]
    c = Cache("f16", 1, 8, 16, 2, 64, False, 1).fill(lens, rng, grid)
    pos = list(range(50))
    q, k, v = normal(rng, (50, 4, 64)), normal(rng, (50, 2, 64)), normal(rng, (50, 2, 64))
    append(c, 0, "f32", q, k, v, [0] * 50, pos, np.zeros(32), 0)
    one = c.download("k"), c.download("v")
    table = D(np.stack([np.ones((50, 32)), np.zeros((50, 32))], -1).astype(np.float32))
    dq, dk, dv, do, ds, dp = D(q), D(k), D(v), D(q), ints([0] * 50), ints(pos)
    lib.gsdh_paged_rope_store(None, c.at, 0, p(dq), 256, p(dk), 128, p(dv), 128, p(do), 256, p(ds), p(dp), 50, 4, p(table), 50, 0)
    assert np.array_equal(one[0], c.download("k")) and np.array_equal(one[1], c.download("v"))
    assert angles(1, 64).shape == (1, 32, 2)


def test_replayed(lib):
    """A captured call reads positions when it runs."""
    rng = np.random.default_rng(8)
    q, f = normal(rng, (6, 2, 64)), frequencies(lib, 64)
    d, r = rope(f, 0)
    dx, do, dp = D(q), D(np.zeros_like(q)), ints([0] * 6)
    st, ge = ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(st))
    lib.gsdh_stream_begin_capture(st)
    lib.gsdh_rope_rows(st, ctypes.byref(r), p(dx), 0, 128, p(do), 128, p(dp), 6, 2, 64)
    lib.gsdh_stream_end_capture(st, ctypes.byref(ge))
    for k in range(4):
        pos = rng.integers(0, 5000, 6).astype(np.int32)
        lib.gsdh_memcpy_h2d(dp.ptr, pos.ctypes.data_as(ctypes.c_void_p), pos.nbytes, None)
        lib.gsdh_stream_sync(None)
        lib.gsdh_graph_replay(ge, st)
        lib.gsdh_stream_sync(st)
        got = H(do, np.float32, q.size).reshape(q.shape).astype(np.float64)
        want, mag = turn(q, f, pos, 0)
        within(got, want, mag, HALF["f32"], 0)
        assert np.array_equal(got, run_rows(lib, q, "f32", f, pos, 0))
    lib.gsdh_graph_destroy(ge)
    lib.gsdh_stream_destroy(st)
