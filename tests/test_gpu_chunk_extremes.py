"""gsdh_paged_chunk_attention where single numbers are extreme: rows near the
largest finite bf16, V there too, scores and scales beyond fp32's range, and the bits
that weights keep."""
import numpy as np
import pytest

from chunk_util import HALF, STEP, attend_chunks, chunk_cache, rounded, run_chunks
from gpu_util import banner
from paged_util import grid, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def eight_bits(rng, shape, exponent):
    """2^exponent .. (2 - 2^-7) 2^exponent: of 127, the largest finite bf16 is among them."""
    return ((128 + rng.integers(0, 128, shape)) * 2.0 ** (exponent - 7)).astype(np.float32)


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("n,m", [(200, 70), (6000, 3), (6000, 40)])
@pytest.mark.parametrize("k,q,scale", [(127, 127, 0.125), (127, 127, -0.125), (127, 117, 1.0), (127, 120, 2.0 ** -100), (120, 127, 3e38),
                                       (-124, 127, 2.0 ** -8), (-118, 120, 2.0 ** -7), (-100, 127, 2.0 ** -31), (127, -126, 2.0 ** -5)])
def test_rows_at_the_end_of_bf16(lib, rows, n, m, k, q, scale, few_rows):
    """Rows of one sign up to the largest bf16.  The products of such rows and their sums are exact in fp32 (16 bits each,
    64 of them), but where they fall below 2^-126 once q's largest element is scaled to 2^-10: a step of 2^-149 is one of
    2^(q - 138) of the products then, and of 64 sums each is off by half of it at most.  Scaling and exponential: 8 half
    steps of the score, as anywhere, where scores do not differ by 100 or more (then there is one weight)."""
    banner(f"chunks bf16 {rows}: K 2^{k}, q 2^{q}, scale {scale:.3g}, {m} of {n}")
    rng, hd = np.random.default_rng(n + m + k + q), 64
    c = chunk_cache("bf16", [n], 16, 1, hd, False, rng, grid, few_rows=few_rows)
    c.set_values(0, 0, 0, np.arange(n), eight_bits(rng, (n, 1, hd), k))
    c.upload()
    qs, scale = eight_bits(rng, (m, 2, hd), q), float(np.float32(scale))
    got = run_chunks(c, 0, qs, rows, [0], [0, m], scale)
    want, mag, top, _, seen, _ = attend_chunks(c, 0, qs, [0], [0, m], scale)
    kk, apart = c.values(0, 0, 0, np.arange(n))[:, 0], True
    for t in range(m):
        for h in range(2):
            x = np.sort(kk[:n - m + t + 1] @ qs[t, h].astype(np.float64) * scale)
            apart &= len(x) == 1 or x[-1] - x[x < x[-1]].max() > 100
    steps = seen * 5 / 8 + 160 + (0 if apart else 16 * top)
    small = 2 * 64 * 2.0 ** (q - 139) * scale if k < -100 else 0.0
    bound = (STEP * steps + small)[..., None] * mag
    if rows == "bf16":
        bound += HALF[rows] * (mag + np.abs(want)) * 1.01
    assert np.isfinite(got).all()
    assert apart or top.max() < 1e4
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("q,scale", [(126, 2.0 ** 20), (126, -2.0 ** 20), (127, 2.0 ** 100), (100, 2.0 ** 100)])
def test_scores_beyond_fp32(lib, kind, q, scale, few_rows):
    """fp32 rows and scales whose product passes fp32's range: the largest score has all the weight."""
    banner(f"chunks {kind} f32: q 2^{q}, scale {scale:.3g}")
    rng, hd, n, m = np.random.default_rng(q), 64, 300, 70
    c = chunk_cache(kind, [n], 16, 1, hd, False, rng, grid, few_rows=few_rows)
    qs = grid(rng, (m, 2, hd)) * np.float32(2.0 ** (q - 1))
    got = run_chunks(c, 0, qs, "f32", [0], [0, m], scale)
    want, mag, _, _, seen, _ = attend_chunks(c, 0, qs, [0], [0, m], scale)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= STEP * (seen * 5 / 8 + 160)[..., None] * mag + 1e-30).all()


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_sums_of_the_largest_v(lib, rows, few_rows):
    """Rows whose scores are all alike, and far from 0, average V rows of the largest finite bf16: that value, although
    the weights of a row, all off by one factor, add up to nearly all that their place leaves them."""
    banner(f"chunks bf16 {rows}: the largest V")
    rng, hd, n, m = np.random.default_rng(1), 64, 1023, 60
    most = (2 - 2.0 ** -7) * 2.0 ** 127
    c = chunk_cache("bf16", [n], 16, 1, hd, False, rng, lambda r, s: np.ones(s, np.float32), few_rows=few_rows)
    c.set_values(1, 0, 0, np.arange(n), np.full((n, 1, hd), most, np.float32))
    c.upload()
    q = np.zeros((m, 16, hd), np.float32)
    q[:, :, 0] = (128 + rng.integers(0, 50, (m, 16))) * 4096.0   # (scores of 5.2e5 to 7.2e5: up to 2^19.99 as exponents of 2)
    got = run_chunks(c, 0, q, rows, [0], [0, m], 1.0)
    assert np.isfinite(got).all()
    assert np.abs(got / most - 1).max() <= STEP * (n * 5 / 8 + 160) + (2.02 * HALF[rows] if rows == "bf16" else 0)


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind,rows", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16"), ("e4m3", "bf16")])
def test_one_position_is_its_v(lib, kind, rows, few_rows):
    """16-bit rows that see one position, whose rounded weight is any of 16 bits, give its V row: weight and sum are the
    same number, and what the quotient and two products round in fp32 is far below half a step of the row."""
    banner(f"chunks {kind} {rows}: one position")
    rng, hd, n = np.random.default_rng(3), 64, 1000
    c = chunk_cache(kind, [n], 16, 1, hd, False, rng, normal, few_rows=few_rows)
    q = rounded(normal(rng, (n, 4, hd)) * np.float32(2.0 ** 12), rows).astype(np.float32)
    got = run_chunks(c, 0, q, rows, [0], [0, n], 1.0, window=1)
    assert np.array_equal(got, np.repeat(c.values(1, 0, 0, np.arange(n)), 4, 1))


@pytest.mark.parametrize("few_rows", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
def test_bits_of_a_weight(lib, kind, few_rows):
    """Rows that see one position give its V row: (a + b) V / l, a + b the 16-bit parts of the weight l, whose bits are any
    (the exponent's rounding is not that of the product).  Off by what the parts leave of l, 2^-23 (a rounded to 11 bits
    leaves 2^-11 of its power of two, b half of its own last bit, 2^-12 of that; three bf16 parts leave nothing), by one
    rounding of the sum (two of three parts), of 1 / l and of the product: five half steps."""
    banner(f"chunks {kind}: bits of a weight")
    rng, hd, n = np.random.default_rng(2), 64, 1000
    c = chunk_cache(kind, [n], 16, 1, hd, False, rng, normal, few_rows=few_rows)
    q = normal(rng, (n, 4, hd)) * np.float32(2.0 ** 14)
    got = run_chunks(c, 0, q, "f32", [0], [0, n], 1.0, window=1)
    want = np.repeat(c.values(1, 0, 0, np.arange(n)), 4, 1)
    off = np.abs(got - want) / np.where(want == 0, 1, np.abs(want)) / STEP
    assert off.max() <= 5.001, off.max()
