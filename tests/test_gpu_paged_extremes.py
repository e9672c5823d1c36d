"""gsdh_paged_attention where single numbers are extreme: NaN and infinities
that only a weight of zero meets."""
import numpy as np
import pytest

from gpu_util import banner
from paged_util import Cache, grid, nan_bits

pytestmark = pytest.mark.gpu
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
