"""gsdh_rope_frequencies at the ends of its arguments: what would give a frequency that is
infinite or no number is refused, and the caller's buffer stays as it was."""
import os

import numpy as np
import pytest

from gsdlq import build, hip

pytestmark = pytest.mark.skipif(not os.path.exists(build.HIP_LIB), reason="engine library not built")
INF = float("inf")


def frequencies(kind, theta=1e6, rd=64, factor=8.0, context=8192.0, low=1.0, high=4.0):
    f = np.full(rd // 2, -7.0)
    try:
        hip.lib().gsdh_rope_frequencies(hip.ROPE_KINDS[kind], theta, rd, factor, context, low, high, hip.ptr(f))
    except hip.HipError:
        assert (f == -7).all()
        raise
    return f


@pytest.mark.parametrize("kind,other", [
    ("by_parts", dict(low=-INF)), ("by_parts", dict(high=INF, context=INF)), ("by_parts", dict(low=-INF, high=INF)), ("plain", dict(theta=1e-320)),
    ("linear", dict(factor=1e-310)), ("ntk", dict(factor=1e-320)), ("ntk", dict(theta=1e300, factor=1e20)), ("by_parts", dict(factor=1e-310))])
def test_refused(kind, other):
    with pytest.raises(hip.HipError, match="frequenc"):
        frequencies(kind, **other)


@pytest.mark.parametrize("kind,other", [
    ("by_parts", dict(high=INF)), ("by_parts", dict(context=INF)), ("by_parts", dict(context=1e-300)), ("plain", dict(theta=1e300)), ("plain", dict(theta=0.5)),
    ("linear", dict(factor=1e300)), ("ntk", dict(factor=0.5))])
def test_given(kind, other):
    f = frequencies(kind, **other)
    assert np.isfinite(f).all() and (f > 0).all()
    if other == dict(high=INF):     # nothing makes so many turns: all are divided
        assert np.allclose(f, frequencies("linear"), rtol=1e-13)
    if other == dict(context=INF):  # everything does
        assert np.allclose(f, frequencies("plain"), rtol=1e-13)
