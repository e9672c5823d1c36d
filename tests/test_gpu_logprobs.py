"""gsdh_token_logprobs against log-softmax in 64 bits.

Tolerances: ln sum is off by the sum's depth (32 or 8 terms a thread, 6 + 2
joins, up to 128 segments: at most 200 half steps of fp32) and the exponentials'
arguments (|x - m| <= 110 where e^(x - m) counts: 110 * 1.45 half steps each,
weighted by p, so at most that), plus four steps of the logarithm; x - m and the
difference add a step of the result.  Entropy: the same for ln s, and for t / s,
whose terms p |x - m| sum to the entropy plus ln s."""
import ctypes

import numpy as np
import pytest

from gpu_util import D, H, banner, p
from paged_util import decode, encode

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()     # raises when no GPU is visible
    return hip.lib()


def bits_of(x, kind):
    return x.astype(np.float32) if kind == "f32" else encode(x, kind)


def call(lib, bits, kind, n, vocab, stride, tokens, top, offset=0, ws=None, entropy=True, stream=None):
    """`bits` flat, the first row `offset` elements in; outputs have a canary behind them."""
    from gsdlq import hip
    es = bits.dtype.itemsize
    dx = D(bits)
    ws = ws or D(np.zeros(lib.gsdh_token_logprobs_workspace_bytes(n, vocab, top), np.uint8))
    lp, en = D(np.full(n + 3, 9.0, np.float32)), D(np.full(n + 3, 9.0, np.float32))
    ids, tl = D(np.full(n * top + 3, -9, np.int32)), D(np.full(n * top + 3, 9.0, np.float32))
    tk = None if tokens is None else D(np.asarray(tokens, np.int32))
    lib.gsdh_token_logprobs(stream, ctypes.c_void_p(dx.ptr.value + offset * es), hip.LOGIT_TYPES[kind], stride, n, vocab, p(tk), top,
                            p(lp) if tk else None, p(en) if entropy else None, p(ids) if top else None, p(tl) if top else None,
                            p(ws), ws.nbytes)
    if stream is not None:
        lib.gsdh_stream_sync(stream)
    lp, en, tl = (H(b, np.float32, k + 3) for b, k in ((lp, n), (en, n), (tl, n * top)))
    ids = H(ids, np.int32, n * top + 3)
    assert (lp[n:] == 9).all() and (en[n:] == 9).all() and (tl[n * top:] == 9).all() and (ids[n * top:] == -9).all()
    return lp[:n], en[:n], ids[:n * top].reshape(n, top), tl[:n * top].reshape(n, top)


def check(x, tokens, got, top):
    """x float64 [n, vocab] of the type's values; rows without a distribution give NaN."""
    lp, en, ids, tl = got
    for r in range(len(x)):
        y = x[r]
        order = np.lexsort((np.arange(len(y)), -np.where(np.isnan(y), -np.inf, y)))[:top]
        assert np.array_equal(ids[r], order), (r, ids[r], order)
        if np.isnan(y).any() or (y == np.inf).any() or not np.isfinite(y).any():
            assert np.isnan(en[r]) and np.isnan(tl[r]).all()
            assert tokens is None or (lp[r] == 0 if tokens[r] == -1 else np.isnan(lp[r]))
            continue
        m = y.max()
        d = y[np.isfinite(y)] - m
        e = np.exp(d)
        s = e.sum()
        spread = float((e * np.minimum(-d, 110)).sum() / s)
        eps = STEP * (200 + 1.45 * spread + 8)

        def near(a, b):
            return np.abs(a - b) <= eps + 3 * STEP * np.abs(b) if np.isfinite(b) else a == b

        if tokens is not None:
            t = tokens[r]
            if t == -1:
                assert lp[r] == 0
            elif not 0 <= t < len(y):
                assert np.isnan(lp[r])
            else:
                assert near(lp[r], y[t] - m - np.log(s)), (r, lp[r], y[t] - m - np.log(s))
        h = np.log(s) - float((e * d).sum() / s)
        assert abs(en[r] - h) <= eps + STEP * 210 * (h + np.log(s)), (r, en[r], h)
        for a, i in zip(tl[r], order):
            assert near(a, y[i] - m - np.log(s)), (r, a, y[i] - m - np.log(s))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab,pad,offset,top", [
    (1, 1, 0, 0, 1), (3, 2, 0, 1, 2), (5, 5, 3, 0, 5), (2, 63, 0, 3, 7), (4, 255, 1, 0, 32), (2, 256, 0, 0, 32), (3, 257, 5, 2, 1),
    (2, 2047, 0, 1, 20), (2, 2048, 8, 0, 20), (3, 2049, 1, 5, 20), (2, 8192, 0, 0, 5), (2, 8193, 0, 7, 32), (1, 32768, 0, 0, 5),
    (7, 40001, 2, 1, 0), (2, 130001, 7, 0, 32), (700, 512, 0, 0, 3), (520, 8185, 0, 0, 20), (513, 8200, 1, 0, 2), (300, 17001, 3, 2, 20)])
def test_sizes(lib, kind, n, vocab, pad, offset, top):
    banner(f"logprobs {kind} {n} x {vocab} (+{pad}, from {offset}) top {top}")
    rng = np.random.default_rng(n * vocab + top)
    stride = vocab + pad
    x = rng.standard_normal(offset + n * stride) * 3
    x[rng.random(len(x)) < 0.02] = -np.inf
    x[rng.random(len(x)) < 4 / vocab] += 9
    rows = x[offset:].reshape(n, stride)
    rows[:, vocab:] = np.nan   # what lies between the rows is not theirs
    rows[:, 0] = 0.5
    x[:offset] = np.nan
    bits = bits_of(x, kind)
    tokens = [int(t) for t in rng.integers(0, vocab, n)]
    tokens[0] = vocab - 1
    if n > 2:
        tokens[1], tokens[2] = -1, vocab
    got = call(lib, bits, kind, n, vocab, stride, tokens, top, offset)
    values = bits.astype(np.float64) if kind == "f32" else decode(bits, kind)
    check(values[offset:].reshape(n, stride)[:, :vocab], tokens, got, top)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 5000, 8192, 70000])
def test_orders_and_ties(lib, kind, vocab):
    """Rows that a selection finds hard: all equal, rising, falling, many ties at
    the border, the largest at one thread's places, signed zeros."""
    banner(f"logprobs {kind} {vocab}: ties and orders")
    rng = np.random.default_rng(vocab)
    ramp = np.arange(vocab, dtype=np.float64)
    spikes = np.zeros(vocab)
    spikes[::1024] = 5 + rng.random(len(spikes[::1024]))
    few = np.zeros(vocab)
    few[rng.integers(0, vocab, 10)] = 1
    zeros = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x = np.stack([np.zeros(vocab), ramp / vocab * 20, -ramp / vocab * 20, spikes, few, zeros, np.round(rng.standard_normal(vocab)),
                  np.where(ramp == vocab - 1, 3.0, -np.inf), np.full(vocab, -7e4), np.where(ramp % 4 == 3, 1.0, 0.0)])
    bits = bits_of(x, kind)
    values = bits.astype(np.float64) if kind == "f32" else decode(bits, kind)
    tokens = [int(t) for t in rng.integers(0, vocab, len(x))]
    for top in (1, 20, 32):
        got = call(lib, bits.reshape(-1), kind, len(x), vocab, vocab, tokens, top)
        check(values, tokens, got, top)
        again = call(lib, bits.reshape(-1), kind, len(x), vocab, vocab, tokens, top)
        for a, b in zip(got, again):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("kind,vocab", [("f32", 700), ("f16", 40000), ("bf16", 9000)])
def test_rows_without_a_distribution(lib, kind, vocab):
    banner(f"logprobs {kind} {vocab}: NaN and infinities")
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((7, vocab))
    x[1, vocab // 2] = np.nan
    x[2, vocab - 1] = np.inf
    x[3] = -np.inf
    x[4] = np.nan
    x[5, 1:] = -np.inf
    x[6, :-1] = -np.inf
    x[6, 0] = np.nan
    bits = bits_of(x, kind)
    values = bits.astype(np.float64) if kind == "f32" else decode(bits, kind)
    tokens = [0, 0, vocab - 1, 0, -1, 0, 0]
    check(values, tokens, call(lib, bits.reshape(-1), kind, 7, vocab, vocab, tokens, 4), 4)


@pytest.mark.parametrize("kind,lowest", [("f32", -3.4028234663852886e38), ("bf16", -3.3895313892515355e38), ("f16", -65504.0)])
@pytest.mark.parametrize("vocab", [100, 9001, 40000])
def test_lowest_values_as_masks(lib, kind, lowest, vocab):
    """Masks of the type's lowest value: all of a row, all but some, mixed with -inf; few allowed tokens."""
    banner(f"logprobs {kind} {vocab}: masks of {lowest:.3g}")
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((6, vocab))
    x[0] = lowest
    x[1, 3:] = lowest
    x[2, ::2] = lowest
    x[3, 7:] = -np.inf
    x[4] = np.where(rng.random(vocab) < 0.5, lowest, -np.inf)
    x[5, : vocab - 2] = lowest
    bits = bits_of(x, kind)
    values = bits.astype(np.float64) if kind == "f32" else decode(bits, kind)
    tokens = [0, 1, 1, 2, -1, vocab - 1]
    tokens[4] = int(np.flatnonzero(np.isfinite(values[4]))[0])
    check(values, tokens, call(lib, bits.reshape(-1), kind, 6, vocab, vocab, tokens, 20), 20)


def test_optional_outputs(lib):
    banner("logprobs: without tokens, entropy or alternatives")
    x = np.random.default_rng(1).standard_normal((3, 9000)).astype(np.float32)
    full = call(lib, x.reshape(-1), "f32", 3, 9000, 9000, [1, 2, 3], 2)
    part = call(lib, x.reshape(-1), "f32", 3, 9000, 9000, None, 2, entropy=False)
    assert (part[0] == 9).all() and (part[1] == 9).all()
    assert np.array_equal(part[2], full[2]) and np.array_equal(part[3], full[3])
    part = call(lib, x.reshape(-1), "f32", 3, 9000, 9000, [1, 2, 3], 0)
    assert np.array_equal(part[0], full[0]) and np.array_equal(part[1], full[1])


def test_workspace_serves_fewer_rows(lib):
    """One workspace: all rows, few (more segments each), all again; nothing behind it is written."""
    banner("logprobs: one workspace, other numbers of rows")
    rng = np.random.default_rng(2)
    n, vocab, top = 600, 9000, 20
    x = rng.standard_normal((n, vocab)).astype(np.float32)
    tokens = [int(t) for t in rng.integers(0, vocab, n)]
    need = lib.gsdh_token_logprobs_workspace_bytes(n, vocab, top)
    for few in (1, 5, 255, 256, 599):
        assert lib.gsdh_token_logprobs_workspace_bytes(few, vocab, top) <= need
    ws = D(np.concatenate([np.zeros(need, np.uint8), np.full(4096, 0xA5, np.uint8)]))
    ws.nbytes = need
    for k in (n, 3, 255, 1, n, 256, 1, n):
        got = call(lib, x[:k].reshape(-1), "f32", k, vocab, vocab, tokens[:k], top, ws=ws)
        check(x[:min(k, 20)].astype(np.float64), tokens, [g[:20] for g in got], top)
        fresh = call(lib, x[:k].reshape(-1), "f32", k, vocab, vocab, tokens[:k], top)
        for a, b in zip(got, fresh):
            assert np.array_equal(a, b)
    ws.nbytes = need + 4096
    assert (H(ws, np.uint8)[need:need + 4096] == 0xA5).all()


def test_captured_and_two_streams(lib):
    banner("logprobs: a captured call, two streams")
    rng = np.random.default_rng(3)
    from gsdlq import hip
    n, vocab, top = 2, 33000, 5
    sets, streams = [], []
    for s in range(2):
        h = ctypes.c_void_p()
        lib.gsdh_stream_create(ctypes.byref(h))
        streams.append(h)
        sets.append(dict(x=D(np.zeros((n, vocab), np.float32)), t=D(np.zeros(n, np.int32)), lp=D(np.zeros(n, np.float32)),
                         en=D(np.zeros(n, np.float32)), ids=D(np.zeros((n, top), np.int32)), tl=D(np.zeros((n, top), np.float32)),
                         ws=D(np.zeros(lib.gsdh_token_logprobs_workspace_bytes(n, vocab, top), np.uint8))))

    def issue(h, b):
        lib.gsdh_token_logprobs(h, p(b["x"]), hip.LOGIT_TYPES["f32"], vocab, n, vocab, p(b["t"]), top, p(b["lp"]), p(b["en"]), p(b["ids"]),
                                p(b["tl"]), p(b["ws"]), b["ws"].nbytes)

    graphs = []
    for h, b in zip(streams, sets):
        g = ctypes.c_void_p()
        lib.gsdh_stream_begin_capture(h)
        issue(h, b)
        lib.gsdh_stream_end_capture(h, ctypes.byref(g))
        graphs.append(g)
    for _ in range(4):
        xs = rng.standard_normal((2, n, vocab)).astype(np.float32)
        ts = rng.integers(0, vocab, (2, n)).astype(np.int32)
        for b, x, t in zip(sets, xs, ts):
            for buf, a in ((b["x"], x), (b["t"], t)):
                a = np.ascontiguousarray(a)
                lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
            lib.gsdh_stream_sync(None)
        for _ in range(5):
            for g, h in zip(graphs, streams):
                lib.gsdh_graph_replay(g, h)
        for h, b, x, t in zip(streams, sets, xs, ts):
            lib.gsdh_stream_sync(h)
            got = (H(b["lp"], np.float32, n), H(b["en"], np.float32, n), H(b["ids"], np.int32, n * top).reshape(n, top),
                   H(b["tl"], np.float32, n * top).reshape(n, top))
            check(x.astype(np.float64), list(t), got, top)
            eager = call(lib, x.reshape(-1), "f32", n, vocab, vocab, list(t), top)
            for a, e in zip(got, eager):
                assert np.array_equal(a, e)
    for g, h in zip(graphs, streams):
        lib.gsdh_graph_destroy(g)
        lib.gsdh_stream_destroy(h)


def test_agrees_with_the_greedy_step(lib):
    """The first alternative is the token that gsdh_greedy_argmax picks."""
    banner("logprobs against the greedy step")
    rng = np.random.default_rng(4)
    for vocab in (512, 32768):
        x = np.round(rng.standard_normal(vocab) * 2, 1).astype(np.float32)   # (ties among the largest)
        dx, t, m = D(x), D(np.zeros(1, np.int32)), D(np.zeros(1, np.float32))
        lib.gsdh_greedy_argmax(None, p(dx), vocab, p(t), p(m))
        _, _, ids, tl = call(lib, x, "f32", 1, vocab, vocab, [0], 2)
        assert ids[0, 0] == H(t, np.int32, 1)[0]
        assert abs((tl[0, 0] - tl[0, 1]) - H(m, np.float32, 1)[0]) < 1e-5
