"""gsdh_paged_attention where single numbers are extreme: NaN and infinities
that only a weight of zero meets, scores far beyond what fp32 tells apart by
one, rows near the ends of the cache type's range."""
import numpy as np
import pytest

from gpu_util import banner
from paged_util import Cache, grid, nan_bits, normal

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24
INF = {"f16": np.uint16(0x7C00), "bf16": np.uint16(0x7F80)}


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def one_hot(kind, n, at, hd=64, heads=2):
    """A sequence of n positions whose position `at` scores 200 (weight 1, the others e^-200: zero in fp32)."""
    rng = np.random.default_rng(n + at)
    c = Cache(kind, 1, -(-n // 16) + 3, 16, 1, hd, False, 1).fill([n], rng, lambda r, s: grid(r, s) * 0)
    c.set_values(1, 0, 0, np.arange(n), grid(rng, (n, 1, hd)))
    k = np.zeros((n, 1, hd), np.float32)
    k[at, 0, 5] = 2.0
    c.set_values(0, 0, 0, np.arange(n), k)
    q = np.zeros((1, heads, hd), np.float32)
    q[0, :, 5] = 100.0
    return c, q


@pytest.mark.parametrize("kind,what", [("f16", "nan"), ("f16", "inf"), ("bf16", "nan"), ("bf16", "inf"), ("e4m3", "nan")])
@pytest.mark.parametrize("at,places", [(0, (20, 700, 4100, 8190)), (8191, (0, 1000, 8100)), (4000, (3999, 3, 6000))])
def test_bad_v_under_a_weight_of_zero(lib, kind, what, at, places):
    """0 * NaN is NaN wherever the row is split: the element of V shows in its
    dim, and in no other, also where its part of the row has no weight."""
    banner(f"paged attention {kind}: V {what} far below the largest score at {at}")
    n, dim = 8192, 9
    c, q = one_hot(kind, n, at)
    v = c.values(1, 0, 0, [at])[0, 0].copy()
    clean = (c.k.copy(), c.v.copy())
    for place in places:
        c.k, c.v = clean[0].copy(), clean[1].copy()
        i = c.rows(None, 0, [place], c.tables[0])
        row = c.v[i]
        row[..., dim] = nan_bits((), kind) if what == "nan" else INF[kind]
        c.v[i] = row
        c.upload()
        got = c.run_attend(0, q, [0], 1.0)[0]
        assert not np.isfinite(got[:, dim]).any(), place
        if what == "nan":
            assert np.isnan(got[:, dim]).all(), place
        rest = np.arange(64) != dim
        # (the one weight: its parts carry 22 bits, its sum and quotient a step each)
        assert (np.abs(got[:, rest] - v[rest]) <= 2.0 ** -21 * np.abs(v[rest])).all(), place
        assert c.status() == 0


def bound(mag, lens):
    """Of outputs whose scores are exact: n / 128 + 96 steps of the sums (as in the attention's own tests)."""
    return STEP * (np.asarray(lens)[:, None, None] / 128 + 96) * mag + 1e-30


@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("exponent", [13, 20, 23, 26, 30, 40])
@pytest.mark.parametrize("scale", [1.0, 0.11])
def test_large_scores(lib, kind, exponent, scale):
    """Scores of 1e4 to 1e13: one position has all the weight, or several with
    the very same score share it (different scores are 2^exponent / 16 * scale
    apart at least, 56 in the smallest case; their products are exact)."""
    banner(f"paged attention {kind}: q around 2^{exponent}, scale {scale}")
    rng = np.random.default_rng(exponent)
    lens = [1, 1, 2, 33, 300, 5000, 1]
    c = Cache(kind, 1, sum(-(-n // 16) for n in lens), 16, 2, 64, False, len(lens), 320,
              scales=np.ones((2, 1, 2), np.float32) if kind == "e4m3" else None).fill(lens, rng, grid)
    q = grid(rng, (len(lens), 16, 64)) * np.float32(2.0 ** exponent)
    got = c.run_attend(0, q, range(len(lens)), scale)
    want, mag, top, _ = c.attend(0, q, range(len(lens)), np.float32(scale))
    assert top.max() > 2.0 ** exponent * scale
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound(mag, lens)).all()
    for i, n in enumerate(lens):
        if n == 1:   # the only position's V row
            v = c.values(1, 0, i, [0])[0]
            assert (np.abs(got[i].reshape(2, 8, 64) - v[:, None]) <= 2.0 ** -21 * np.abs(v[:, None])).all()


@pytest.mark.parametrize("k,q,v,scale", [
    (0, 0, 110, 0.11), (0, 0, 126, 0.11), (0, 0, -60, 0.11),       # V near both ends of the type
    (120, -120, 0, 0.11), (124, -124, 124, 0.11),                   # K as large, with a q as small
    (120, 0, 0, 0.11 * 2.0 ** -120), (126, -6, 126, 0.11 * 2.0 ** -120),   # or a scale as small
    (-100, 100, 0, 0.11), (-60, 60, 60, 0.11), (100, 10, 100, 1.0)])
def test_bf16_rows_over_their_range(lib, k, q, v, scale):
    """bf16 rows have fp32's range: whatever is finite gives the finite average
    that the definition gives (K, q and V are small whole numbers times the powers
    of two given, so that the scores' sums are exact)."""
    banner(f"paged attention bf16: K 2^{k}, q 2^{q}, V 2^{v}, scale {scale:.3g}")
    rng = np.random.default_rng(k + 1000)
    lens = [1, 33, 300, 6000]
    c = Cache("bf16", 1, sum(-(-n // 16) for n in lens), 16, 1, 64, False, len(lens), 400).fill(lens, rng, grid)
    for s, n in enumerate(lens):
        at = np.arange(n)
        c.set_values(0, 0, s, at, grid(rng, (n, 1, 64)) * np.float32(2.0 ** k))
        c.set_values(1, 0, s, at, grid(rng, (n, 1, 64)) * np.float32(2.0 ** v))
    c.upload()
    qs = grid(rng, (len(lens), 4, 64)) * np.float32(2.0 ** q)
    got = c.run_attend(0, qs, range(len(lens)), scale)
    want, mag, top, _ = c.attend(0, qs, range(len(lens)), np.float32(scale))
    assert np.isfinite(got).all()
    # the scores' scaling and their exponential: 8 steps each, twice (in weight and sum), where they do not pick one position
    steps = np.asarray(lens)[:, None] / 128 + 96 + np.where(top < 1e4, 16 * top, 0)
    assert (np.abs(got - want) <= STEP * steps[..., None] * mag + 1e-30).all()


@pytest.mark.parametrize("k", [0, 100, 126])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-42])
def test_bf16_scale_of_zero(lib, k, scale):
    """A scale of 0 (or next to it) weighs all positions alike (nearly), however large K is."""
    banner(f"paged attention bf16: K 2^{k}, scale {scale:.3g}")
    rng = np.random.default_rng(k)
    lens = [1, 40, 3000]
    c = Cache("bf16", 1, sum(-(-n // 16) for n in lens), 16, 1, 64, False, len(lens), 200).fill(lens, rng, grid)
    for s, n in enumerate(lens):
        c.set_values(0, 0, s, np.arange(n), grid(rng, (n, 1, 64)) * np.float32(2.0 ** k))
    c.upload()
    q = grid(rng, (len(lens), 4, 64))
    got = c.run_attend(0, q, range(len(lens)), scale)
    want, mag, top, _ = c.attend(0, q, range(len(lens)), float(np.float32(scale)))
    # (1e-42 times log2 e is rounded to a multiple of 2^-149: half of that to 1.4e-42, of the score, twice)
    steps = np.asarray(lens)[:, None] / 128 + 96 + 16 * top + 2 * top * 2.0 ** -150 / 1.4e-42 / STEP
    assert (np.abs(got - want) <= STEP * steps[..., None] * mag + 1e-30).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_infinite_k(lib, kind):
    """An infinity in K: a score of +inf or NaN leaves no distribution (NaN); one
    of -inf is a weight of 0 (or NaN, where the parts of q differ in sign), and
    a row of nothing else is NaN, not the zeros of an empty sequence."""
    banner(f"paged attention {kind}: infinities in K")
    rng = np.random.default_rng(21)
    lens, at, dim = [300, 300, 5000, 1, 1, 40, 0], [7, 299, 4000, 0, 0, None, None], 11
    c = Cache(kind, 1, sum(-(-n // 16) for n in lens), 16, 1, 64, False, len(lens), 320).fill(lens, rng, grid)
    for s, p in enumerate(at):
        if lens[s]:
            i = c.rows(None, 0, np.arange(lens[s]) if p is None else [p], c.tables[s])
            row = c.k[i]
            row[..., dim] = INF[kind] | (0x8000 if s % 2 else 0)
            c.k[i] = row
    c.upload()
    q = normal(rng, (len(lens), 16, 64))
    got = c.run_attend(0, q, range(len(lens)), 0.1)
    assert (got[6] == 0).all()
    seen = set()
    for s in range(6):
        down = q[s, :, dim] * (-1 if s % 2 else 1) < 0   # heads whose score is -inf
        assert not np.isfinite(got[s][~down]).any(), s
        if at[s] is None or lens[s] == 1:
            assert np.isnan(got[s]).all(), s
            continue
        keep = np.delete(np.arange(lens[s]), at[s])
        k, v = (c.values(w, 0, s, keep)[:, 0] for w in (0, 1))
        for h in np.flatnonzero(down):
            if np.isnan(got[s, h]).all():
                continue
            x = k @ q[s, h].astype(np.float64) * np.float32(0.1)
            e = np.exp(x - x.max())
            e /= e.sum()
            dot = (np.abs(k) @ np.abs(q[s, h])).max() * 0.1
            steps = 2 * ((64 + 16) * dot + 8 * np.abs(x).max()) + lens[s] / 128 + 96
            assert (np.abs(got[s, h] - e @ v) <= STEP * steps * (e @ np.abs(v)) + 1e-30).all(), (s, h)
            seen.add((s, h))
    assert len(seen) > 0
