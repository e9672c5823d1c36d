"""gsdh_paged_chunk_attention where a block goes through more pages than it holds
the indices of at once (256: 31 tiles of 64 positions in pages of 8, 63 in pages of
16, 255 in pages of 64).  A table may name a page many times, so hundreds of
thousands of positions lie over a few hundred pages, and the definition in 64
bits goes by these: a score per row of the pool, its weight times as often as
the table has it."""
import numpy as np
import pytest

from chunk_util import HALF, STEP, run_chunks
from gpu_util import banner
from paged_util import Cache, encode, grid

pytestmark = pytest.mark.gpu
HEADS, KV, TILE = 16, 8, 64


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def long_cache(kind, page, n, hd, head_major, m, first, rng):
    """One sequence of n positions.  Of each of 64 dims two pages have a row that scores 40 with a q of 20 there, each at
    one place of the table between `first` and what the first of m tokens sees; all others score 0."""
    hot, cold = 128, 40
    c = Cache(kind, 1, hot + cold, page, KV, hd, head_major, 1, -(-n // page) + 1)
    k = np.zeros((hot + cold, page, KV, hd), np.float32)
    slots = rng.integers(0, page, hot)
    k[np.arange(hot), slots, :, np.arange(hot) % 64] = 2.0
    v = grid(rng, k.shape)
    for which, x in ((0, k), (1, v)):
        if c.scales is not None:
            x = x / c.scales[which, 0][:, None]
        (c.k, c.v)[which][0] = encode(x if not head_major else x.transpose(0, 2, 1, 3), kind)
    c.lens[0] = n
    used = -(-n // page)
    c.tables[0, :used] = hot + rng.integers(0, cold, used)
    places = rng.choice(np.arange(first // page + 1, (n - m) // page), hot, replace=False)
    c.tables[0, places] = np.arange(hot)
    c.few_rows = False
    c.upload()
    return c, k, v


@pytest.mark.parametrize("kind,rows,hd", [("f16", "f32", 64), ("f16", "f16", 64), ("bf16", "f32", 64), ("bf16", "bf16", 64), ("e4m3", "f32", 64), ("e4m3", "f16", 64),
                                          ("e4m3", "bf16", 64), ("f16", "f32", 128), ("bf16", "f32", 128), ("e4m3", "f32", 128), ("f16", "f16", 256), ("e4m3", "f32", 256)])
@pytest.mark.parametrize("m", [3, 20, 40])   # few rows, one or two waves' of them; many rows
@pytest.mark.parametrize("page,n,window,head_major", [(8, 200003, 0, False), (8, 210001, 150000, True), (16, 300007, 0, True), (64, 1000001, 0, False)])
def test_more_pages_than_are_held(lib, kind, rows, hd, m, page, n, window, head_major):
    from gsdlq import hip
    cus = hip.device_info()[2]
    tiles = (window or n) / (cus // KV) / TILE
    assert tiles > 255 * page / TILE + 1
    banner(f"chunks {kind} {rows} hd {hd}: {m} of {n}, pages of {page}, {tiles:.0f} tiles a block")
    rng = np.random.default_rng(n + m)
    c, k, v = long_cache(kind, page, n, hd, head_major, m, n - window if window else 0, rng)
    q = np.zeros((m, HEADS, hd), np.float32)
    dims = (np.arange(m)[:, None] * HEADS + np.arange(HEADS)) % 64
    np.put_along_axis(q, dims[..., None], 20.0, -1)
    got = run_chunks(c, 0, q, rows, [0], [0, m], 1.0, window)
    times = np.zeros((m, len(k) * page))    # how often a row of the pool is seen
    for t in range(m):
        pos = np.arange(max(0, n - m + t + 1 - window) if window else 0, n - m + t + 1)
        times[t] = np.bincount(c.tables[0, pos // page] * page + pos % page, minlength=len(k) * page)
    worst = 0.0
    for h in range(HEADS):
        kv = h // (HEADS // KV)
        kk, vv = (x[:, :, kv].reshape(-1, hd).astype(np.float64) for x in (k, v))
        w = times * np.exp(q[:, h].astype(np.float64) @ kk.T - 40.0)
        w /= w.sum(1, keepdims=True)
        want, mag = w @ vv, w @ np.abs(vv)
        # (scores of 0 and 40 are exact; 8 half steps of 40 in the weight and in the sum; the sums as in chunk_util.check)
        bound = STEP * (2 * 8 * 40 + n * 5 / 8 + 160) * mag + n * 2.0 * 2.0 ** -38
        if rows != "f32":
            bound += HALF[rows] * (mag + np.abs(want)) * 1.01
        worst = max(worst, (np.abs(got[:, h] - want) / bound).max())
    assert worst <= 1, worst
    assert c.status() == 0
