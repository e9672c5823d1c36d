"""gsdh_paged_attention over rows up to the largest finite bf16, and with scales
whose product with q passes fp32's range."""
import numpy as np
import pytest

from gpu_util import banner
from paged_util import Cache, grid

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def eight_bits(rng, shape, exponent):
    """2^exponent .. (2 - 2^-7) 2^exponent: of 127, the largest finite bf16 is among them."""
    return ((128 + rng.integers(0, 128, shape)) * 2.0 ** (exponent - 7)).astype(np.float32)


@pytest.mark.parametrize("kind,k,q,scale", [
    ("bf16", 127, 127, 0.125), ("bf16", 127, 127, -0.125), ("bf16", 127, 117, 1.0), ("bf16", 127, 120, 2.0 ** -130), ("bf16", 120, 127, 3e38),
    ("bf16", -124, 127, 2.0 ** -8), ("bf16", -118, 120, 2.0 ** -7), ("bf16", -100, 127, 2.0 ** -31), ("bf16", 127, -126, 2.0 ** -5),
    ("f16", 0, 126, 2.0 ** 20), ("f16", 0, 127, -2.0 ** 100), ("e4m3", 0, 126, 2.0 ** 20)])
def test_rows_at_the_end_of_the_range(lib, kind, k, q, scale):
    """Products of rows of 8 bits and their sums are exact in fp32; of scores beyond 2^100 the second largest differs from
    the largest by 2^-14 of it at least, so that it has no weight, whichever parts of the row they lie in."""
    banner(f"paged attention {kind}: K 2^{k}, q 2^{q}, scale {scale:.3g}")
    rng = np.random.default_rng(k + q)
    lens = [1, 32, 31, 5, 300, 6000]
    c = Cache(kind, 1, sum(-(-n // 16) for n in lens), 16, 1, 64, False, len(lens), 400).fill(lens, rng, grid)
    for s, n in enumerate(lens):
        c.set_values(0, 0, s, np.arange(n), eight_bits(rng, (n, 1, 64), k))
    c.upload()
    qs, scale = eight_bits(rng, (len(lens), 4, 64), q), float(np.float32(scale))
    got = c.run_attend(0, qs, range(len(lens)), scale)
    want, mag, top, _ = c.attend(0, qs, range(len(lens)), scale)
    assert np.isfinite(got).all()
    if top.max() > 2.0 ** 100:
        for s, n in enumerate(lens):
            x = np.sort(c.values(0, 0, s, np.arange(n))[:, 0] @ qs[s].T.astype(np.float64) * scale, 0)
            for h in range(4):
                second = x[x[:, h] < x[-1, h], h].max(initial=-np.inf)
                assert x[-1, h] - second > 2.0 ** -14 * abs(x[-1, h])
    steps = np.asarray(lens)[:, None] / 128 + 96 + np.where(top < 1e4, 16 * top, 0)
    assert (np.abs(got - want) <= STEP * steps[..., None] * mag + 1e-30).all()
