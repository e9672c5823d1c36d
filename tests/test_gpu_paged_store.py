"""gsdh_paged_rope_store: the rotation and the stored bits equal the plain form
(fp32 products and sums rounded one by one, then one rounding to the cache's
type), and the one-token append's on the same angles, bit for bit; nothing else
in the pools changes."""
import ctypes

import numpy as np
import pytest

from gpu_util import D, H, banner, p
from paged_util import Cache, angles, encode, ints, normal, rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def _store(c, layer, qkv, heads, seqs, pos, table, interleaved, in_place=False, pad=0):
    """q_out of the call on rows of one buffer, as one projection leaves them; outputs start at 3."""
    n, kv, hd = len(seqs), c.kv, c.hd
    w = (heads + 2 * kv) * hd + pad
    flat = np.zeros((n, w), np.float32)
    flat[:, :(heads + 2 * kv) * hd] = qkv.reshape(n, -1)
    x, out = D(flat), D(np.full((n, heads * hd + 4), 3.0, np.float32))
    at = lambda h: ctypes.c_void_p(x.ptr.value + 4 * h * hd)  # noqa: E731
    qo, stride = (at(0), w) if in_place else (p(out), heads * hd + 4)
    ds, dp, da = ints(seqs), ints(pos), D(table)
    c.lib.gsdh_paged_rope_store(None, c.at, layer, at(0), w, at(heads), w, at(heads + kv), w, qo, stride, p(ds), p(dp), n, heads,
                                p(da), len(table), interleaved)
    if in_place:
        r = H(x, np.float32, n * w).reshape(n, w)
        assert np.array_equal(r.view(np.uint32)[:, heads * hd:], flat.view(np.uint32)[:, heads * hd:])   # K, V, padding as they were
        return r[:, :heads * hd].reshape(n, heads, hd)
    r = H(out, np.float32, n * (heads * hd + 4)).reshape(n, -1)
    assert (r[:, heads * hd:] == 3.0).all()
    return r[:, :heads * hd].reshape(n, heads, hd)


def _expect(c, layer, qkv, heads, seqs, pos, table, interleaved, skipped=()):
    """Stores into the model's pools; q rows as they should come back (3 where nothing is written)."""
    q = np.full((len(seqs), heads, c.hd), 3.0, np.float32)
    for t, (s, x) in enumerate(zip(seqs, pos)):
        if t in skipped:
            continue
        a = table[x][None]
        q[t] = rotate(qkv[t:t + 1, :heads], a, interleaved)[0]
        k, v = rotate(qkv[t:t + 1, heads:heads + c.kv], a, interleaved), qkv[t:t + 1, heads + c.kv:]
        c.set_values(0, layer, s, [x], k)
        c.set_values(1, layer, s, [x], v)
    return q


def _same_pools(c):
    assert np.array_equal(c.download("k"), c.k)
    assert np.array_equal(c.download("v"), c.v)


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd,page,head_major", [(4, 2, 64, 8, False), (32, 8, 128, 16, True), (8, 1, 256, 64, False), (3, 3, 64, 256, True)])
@pytest.mark.parametrize("interleaved", [1, 0])
def test_ragged_tokens(lib, kind, heads, kv, hd, page, head_major, interleaved):
    banner(f"paged store {kind} {heads}/{kv}x{hd} page {page} {'pairs' if interleaved else 'halves'}")
    rng = np.random.default_rng(heads + page)
    lens = [70, 1, 33, 300]
    c = Cache(kind, 2, 90, page, kv, hd, head_major, 4, -(-300 // page) + 1).fill(lens, rng, normal)
    if c.scales is not None:   # (any scale, not only powers of two)
        c.scales = np.exp(rng.uniform(-2, 2, c.scales.shape)).astype(np.float32)
        c.upload()
    todo = [(0, t) for t in range(60, 70)] + [(1, 0), (-1, 5), (3, 299), (3, 0), (2, 32), (3, 128), (-1, -1)]
    seqs, pos = [s for s, _ in todo], [t for _, t in todo]
    qkv = (normal(rng, (len(todo), heads + 2 * kv, hd)) * np.exp(rng.uniform(-8, 5, (len(todo), 1, 1)))).astype(np.float32)
    table = angles(300, hd)
    got = _store(c, 1, qkv, heads, seqs, pos, table, interleaved, pad=8)
    want = _expect(c, 1, qkv, heads, seqs, pos, table, interleaved, skipped=[t for t, s in enumerate(seqs) if s < 0])
    assert np.array_equal(got, want)
    _same_pools(c)
    assert c.status() == 0


def test_in_place_and_special_values(lib):
    """q rotated where it lies; NaN, infinities, halfway and out-of-range values in 8 bits."""
    banner("paged store: in place, special values")
    c = Cache("e4m3", 1, 4, 8, 1, 64, False, 1, 4, scales=np.full((2, 1, 1), 0.5, np.float32)).fill([10], np.random.default_rng(1), normal)
    x = np.zeros((1, 4, 64), np.float32)
    x[0, :2] = normal(np.random.default_rng(2), (2, 64))
    x[0, 3, :16] = [np.nan, np.inf, -np.inf, 224, 232, 240, 1e9, -1e9, 0, -0.0, 0.5 * 2.0 ** -9, 0.5 * 2.0 ** -10, 0.5 * 3 * 2.0 ** -10,
                    0.5 * 1.0625, 0.5 * 1.1875, 0.5 * 2.0 ** -11]
    x[0, 2] = x[0, 3]
    table = np.zeros((10, 32, 2), np.float32)
    table[..., 0] = 1   # no rotation: K' = K
    got = _store(c, 0, x, 2, [0], [9], table, 0, in_place=True)
    assert np.array_equal(got, x[:, :2])
    with np.errstate(invalid="ignore"):
        k = rotate(x[:, 2:3], table[9:10], 0)[0, 0]   # (an infinity's partner is inf * 0)
    for pool, rows in (("k", k), ("v", x[0, 3])):
        row = c.download(pool)[c.rows(None, 0, [9], c.tables[0])][0, 0]
        nan = np.isnan(rows)
        assert nan.any() and ((row[nan] & 127) == 127).all()
        assert np.array_equal(row[~nan], encode(rows / np.float32(0.5), "e4m3")[~nan])


def test_equals_the_one_token_append(lib):
    banner("paged store against gsdh_rope_and_store_kv")
    rng = np.random.default_rng(3)
    heads, kv, hd, ms = 8, 2, 128, 512
    c = Cache("f16", 2, ms // 16, 16, kv, hd, False, 1)
    c.k[:], c.v[:] = 0, 0
    c.tables[0], c.lens[0], c.refs[:] = np.arange(ms // 16), ms, 1
    c.upload()
    libm = ctypes.CDLL("libm.so.6")
    for f in ("powf", "cosf", "sinf"):
        getattr(libm, f).restype = ctypes.c_float
        getattr(libm, f).argtypes = [ctypes.c_float] * (2 if f == "powf" else 1)
    table = np.zeros((ms, hd // 2, 2), np.float32)
    for pos in (0, 7, 300, 511):
        for i in range(hd // 2):
            a = np.float32(pos) * (np.float32(1) / np.float32(libm.powf(1e6, np.float32(2 * i) / np.float32(hd))))
            table[pos, i] = libm.cosf(a), libm.sinf(a)
    for pos in (0, 7, 300, 511):
        for interleaved in (0, 1):
            x = normal(rng, (1, heads + 2 * kv, hd))
            got = _store(c, 1, x, heads, [0], [pos], table, interleaved)
            dq, dk, dv = D(x[0, :heads]), D(x[0, heads:heads + kv]), D(x[0, heads + kv:])
            kc, vc = D(np.zeros_like(c.k)), D(np.zeros_like(c.v))
            lib.gsdh_rope_and_store_kv(None, p(dq), p(dk), p(dv), p(kc), p(vc), 1, pos, heads, kv, hd, ms, 1e6, interleaved)
            assert np.array_equal(got[0].reshape(-1), H(dq, np.float32, heads * hd))
            row = (1, pos // 16, pos % 16)
            for mine, theirs in (("k", kc), ("v", vc)):
                assert np.array_equal(c.download(mine)[row], H(theirs, np.uint16, c.k.size).reshape(c.k.shape)[row])


def test_what_is_left_out(lib):
    """Tokens outside the cache, the sequence or the angles, and rows of shared
    or unheld pages: nothing of them is written, the others are."""
    from gsdlq import hip
    banner("paged store: refused tokens")
    rng = np.random.default_rng(4)
    heads, table = 2, angles(100, 64)
    c = Cache("f16", 1, 30, 8, 2, 64, False, 5, 6).fill([40, 40, 40, 20, 0], rng, normal)
    c.tables[2, 1] = 30
    c.tables[2, 2] = -3
    c.refs[c.tables[1, 2]] = 2
    c.refs[c.tables[1, 3]] = 0
    c.upload()
    index = [(5, 0), (1, 40), (1, -1), (2, 8), (2, 16), (3, 20), (4, 0), (2 ** 30, 3)]
    for todo, bits in ((index, hip.PAGES_BAD_INDEX), ([(1, 16), (1, 31)], hip.PAGES_SHARED)):
        good = [(0, 39), (3, 19), (1, 39)]
        seqs, pos = [s for s, _ in todo + good], [t for _, t in todo + good]
        x = normal(rng, (len(seqs), heads + 4, 64))
        got = _store(c, 0, x, heads, seqs, pos, table, 1)
        want = _expect(c, 0, x, heads, seqs, pos, table, 1, skipped=range(len(todo)))
        assert np.array_equal(got, want)
        _same_pools(c)
        assert c.status() == bits
        c.clear_status()
    # fewer angles than positions
    x = normal(rng, (2, heads + 4, 64))
    got = _store(c, 0, x, heads, [0, 0], [38, 39], table[:39], 1)
    assert np.array_equal(got, _expect(c, 0, x, heads, [0, 0], [38, 39], table, 1, skipped=[1]))
    _same_pools(c)
    assert c.status() == hip.PAGES_BAD_INDEX
    # a caller that counts pages itself gives no refs
    c.clear_status()
    c.c = c.struct(refs=None)
    c.at = ctypes.byref(c.c)
    x = normal(rng, (1, heads + 4, 64))
    _store(c, 0, x, heads, [1], [16], table, 1)
    _expect(c, 0, x, heads, [1], [16], table, 1)
    _same_pools(c)
    assert c.status() == 0


def test_long_prompts(lib):
    """Thousands of tokens of several sequences in one call."""
    banner("paged store: 4099 tokens")
    rng = np.random.default_rng(5)
    lens = [1500, 1300, 1299]
    c = Cache("bf16", 1, 300, 16, 2, 64, True, 3, 100).fill(lens, rng, normal)
    seqs = np.repeat(np.arange(3), lens)
    pos = np.concatenate([np.arange(n) for n in lens])
    order = rng.permutation(len(seqs))
    x = normal(rng, (len(seqs), 4 + 4, 64))
    table = angles(1500, 64)
    got = _store(c, 0, x, 4, seqs[order], pos[order], table, 1)
    a = table[pos[order]]
    assert np.array_equal(got, rotate(x[:, :4], a, 1))
    k = rotate(x[:, 4:6], a, 1)
    for s in range(3):
        mine = seqs[order] == s
        c.set_values(0, 0, s, pos[order][mine], k[mine])
        c.set_values(1, 0, s, pos[order][mine], x[mine, 6:])
    _same_pools(c)
