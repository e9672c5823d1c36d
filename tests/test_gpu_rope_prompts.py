"""gsdh_rope_rows and gsdh_paged_rope_append over the rows of prompts: calls of more
blocks than the chip takes at once, whose threads have four items each, against the
rotation in 64 bits (tolerances as in test_gpu_rope) and, bit for bit, the same rows
in calls of a few tokens; and the append beside the store with a table."""
import numpy as np
import pytest

from chunk_util import HALF, rounded
from gpu_util import D, H, banner, p
from paged_util import Cache, decode, grid, ints, normal
from test_gpu_rope import KV_HALF, LEAST, append, frequencies, run_rows, turn, within

pytestmark = pytest.mark.gpu
THREADS, BLOCKS = 256, 2048   # items of a block, blocks up to which a thread has one item


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()
    return hip.lib()


def blocks(heads, kv, hd, rd):
    """Of one token with an item per thread (tokens of up to half a block's items share one)."""
    items = (heads + kv) * (-(-rd // 2 // 4) + -(-(hd - rd) // 8)) + kv * (hd // 8)
    assert items > THREADS // 2
    return -(-items // THREADS)


# items of a token: 640, 160 (at the switch and behind it), 1377 (two blocks of four items per thread), 153, 1056, 2048
ROWS = [(40, 128, 128, 683), (10, 128, 128, 2048), (10, 128, 128, 2049), (81, 128, 50, 420), (9, 128, 20, 2050), (88, 96, 96, 411), (16, 1024, 1024, 300)]


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("heads,hd,rd,n", ROWS)
def test_rows_of_a_prompt(lib, rows, interleaved, heads, hd, rd, n):
    assert (n * blocks(heads, 0, hd, rd) > BLOCKS) == (n != 2048)
    banner(f"rope {rows} {n} x {heads}x{hd} of {rd} {'pairs' if interleaved else 'halves'}")
    rng = np.random.default_rng(heads + rd)
    pos = rng.integers(-2000, 200000, n)
    f = frequencies(lib, rd)
    q = rounded(normal(rng, (n, heads, hd)), rows).astype(np.float32)
    want, mag = turn(q, f, pos, interleaved, 1.25)
    got = run_rows(lib, q, rows, f, pos, interleaved, 1.25, pad=8, out_pad=16)
    within(got, want, mag, HALF[rows], LEAST[rows])
    assert np.array_equal(got[..., rd:], q[..., rd:])
    assert np.array_equal(got, run_rows(lib, q, rows, f, pos, interleaved, 1.25, in_place=True, pad=8))
    for t in (0, n // 2, n - 12):
        assert np.array_equal(got[t:t + 12], run_rows(lib, q[t:t + 12], rows, f, pos[t:t + 12], interleaved, 1.25))


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,rd,interleaved,page,head_major,lens", [
    (32, 8, 128, 128, 1, 16, False, [500, 1, 230]), (12, 4, 64, 64, 0, 64, True, [1200, 900]), (64, 8, 128, 20, 0, 32, True, [300, 77, 30]),
    (25, 5, 256, 250, 1, 8, False, [250, 170])])
def test_prompts_into_the_cache(lib, kind, rows, heads, kv, hd, rd, interleaved, page, head_major, lens):
    """All positions of some sequences in any order, padding and bad tokens among them; nothing else in the pools changes."""
    from gsdlq import hip
    rng = np.random.default_rng(heads + page)
    c = Cache(kind, 2, sum(-(-n // page) for n in lens) + 4, page, kv, hd, head_major, len(lens) + 1, max(lens) // page + 2).fill(lens + [0], rng, grid)
    c.refs[c.tables[0, 2]] = 2       # a page that has two holders
    c.upload()
    seqs = np.repeat(np.arange(len(lens)), lens)
    pos = np.concatenate([np.arange(n) for n in lens])
    order = rng.permutation(len(seqs))
    seqs, pos = seqs[order], pos[order]
    bad = {3: (-1, 5), 700 % len(seqs): (-7, 0), 11: (len(lens) + 1, 0), 300 % len(seqs): (0, lens[0]), 77: (len(lens), 0), len(seqs) - 1: (0, -1)}
    seqs, pos = seqs.copy(), pos.copy()
    for t, (s, x) in bad.items():
        seqs[t], pos[t] = s, x
    n = len(seqs)
    assert n * blocks(heads, kv, hd, rd) > BLOCKS
    banner(f"append {rows} to {kind} {n} x {heads}/{kv}x{hd} of {rd}")
    ok = np.array([t not in bad and not (seqs[t] == 0 and pos[t] // page == 2) for t in range(n)])
    q, k, v = (rounded(2 * normal(rng, (n, h, hd)), rows).astype(np.float32) for h in (heads, kv, kv))
    f = frequencies(lib, rd, "by_parts", 4.0)
    want_q, mag_q = turn(q, f, pos, interleaved, 1.1)
    want_k, mag_k = turn(k, f, pos, interleaved, 1.1)
    before = c.download("k"), c.download("v")
    got = append(c, 1, rows, q, k, v, seqs, pos, f, interleaved, 1.1)
    within(got[ok], want_q[ok], mag_q[ok], HALF[rows], LEAST[rows])
    assert (got[~ok] == 7).all()
    assert c.status() == hip.PAGES_BAD_INDEX | hip.PAGES_SHARED
    pools = c.download("k"), c.download("v")
    scales = np.ones((2, kv)) if c.scales is None else c.scales[:, 1].astype(np.float64)
    for which, (want, mag) in enumerate(((want_k, mag_k), (v.astype(np.float64), np.zeros(v.shape)))):
        written = np.zeros(before[0].shape, bool)
        for s in range(len(lens)):
            mine = ok & (seqs == s)
            at = c.rows(None, 1, pos[mine], c.tables[s])
            written[at] = True
            x, m = want[mine] / scales[which][:, None], mag[mine] / scales[which][:, None]
            limit = 448.0 if kind == "e4m3" else np.inf
            within(decode(pools[which][at], kind), np.clip(x, -limit, limit), m + np.abs(x) * 2.0 ** -3, KV_HALF[kind], LEAST[kind])
        assert np.array_equal(pools[which][~written], before[which][~written])
    # in place, and the same tokens a few at a time
    again = append(c, 1, rows, q, k, v, seqs, pos, f, interleaved, 1.1, in_place=True)
    assert np.array_equal(again[ok], got[ok]) and np.array_equal(again[~ok], q[~ok])
    c.upload()
    for t in range(0, n, 100):
        part = slice(t, t + 100)
        assert np.array_equal(got[part], append(c, 1, rows, q[part], k[part], v[part], seqs[part], pos[part], f, interleaved, 1.1))
    assert all(np.array_equal(a, b) for a, b in zip(pools, (c.download("k"), c.download("v"))))


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_append_is_the_store_on_quarter_turns(lib, kind, interleaved):
    """Frequencies of whole quarter turns per position, another for each pair.  The table's cosines and sines are 0, 1 and
    -1; an angle that fp64 forms is off by less than 2^-44 of a turn, which nothing shows in fp32 beside 1/4 and 1/2, nor
    2 pi 2^-44 of a row's element beside another within twice of it.  So K, V and q are the store's, bit for bit."""
    rng = np.random.default_rng(7)
    n, heads, kv, hd = 60, 4, 2, 64
    c = Cache(kind, 1, 8, 16, kv, hd, False, 1).fill([n], rng, grid)
    pos, quarters = np.arange(n), 1 + np.arange(hd // 2) % 7
    q, k, v = ((rng.uniform(1, 2, (n, h, hd)) * rng.choice([-1, 1], (n, h, hd))).astype(np.float32) for h in (heads, kv, kv))
    got = append(c, 0, "f32", q, k, v, [0] * n, pos, quarters * (np.pi / 2), interleaved)
    one = c.download("k"), c.download("v")
    turns = pos[:, None] * quarters % 4
    table = D(np.stack([np.array([1, 0, -1, 0])[turns], np.array([0, 1, 0, -1])[turns]], -1).astype(np.float32))
    c.upload()
    dq, dk, dv, do, ds, dp = D(q), D(k), D(v), D(q), ints([0] * n), ints(pos)
    w, kw = heads * hd, kv * hd
    lib.gsdh_paged_rope_store(None, c.at, 0, p(dq), w, p(dk), kw, p(dv), kw, p(do), w, p(ds), p(dp), n, heads, p(table), n, interleaved)
    assert np.array_equal(one[0], c.download("k")) and np.array_equal(one[1], c.download("v"))
    assert np.array_equal(got, H(do, np.float32, n * w).reshape(n, heads, hd).astype(np.float64))
    # (it turned: the second half of a turn is the negative of what came)
    half = (turns == 2)[:, None, :]
    i, j = (np.arange(0, hd, 2), np.arange(1, hd, 2)) if interleaved else (np.arange(hd // 2), np.arange(hd // 2, hd))
    for d in (i, j):
        at = np.broadcast_to(half, got[..., d].shape)
        assert at.any() and np.array_equal(got[..., d][at], -q[..., d][at])
