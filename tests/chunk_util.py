"""Rows of the three types on the host, and chunk attention's definition in 64
bits beside its call, over the model cache of paged_util."""
import numpy as np

from gpu_util import D, H, p
from paged_util import Cache, decode, encode

STEP = 2.0 ** -24                       # half a step of fp32, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def row_bits(x, rows):
    """float -> the bits of a row type."""
    return np.asarray(x, np.float32) if rows == "f32" else encode(x, rows)


def row_values(bits, rows):
    return bits.astype(np.float64) if rows == "f32" else decode(bits, rows)


def rounded(x, rows):
    """The values that the type holds."""
    return row_values(row_bits(x, rows), rows)


def space(c, n, tokens, heads):
    return D(np.full(c.lib.gsdh_paged_chunk_attention_workspace_bytes(c.at, n, tokens, heads), 0xA5, np.uint8))   # (may hold anything)


FEW_ROWS, FEW_ROOM = 64, 1024   # mean rows of a chunk up to which, positions of a table from which on a call goes by few rows


def few(c, q, seqs, starts):
    """The same chunks, with padding behind them, as a call that goes by few rows."""
    assert c.width * c.page >= FEW_ROOM
    n = len(starts) - 1
    seqs, starts = list(range(n) if seqs is None else seqs), list(starts)
    more = -(-q.shape[0] * q.shape[1] // c.kv // FEW_ROWS) - n
    return seqs + [-1] * max(more, 0), starts + [starts[-1]] * max(more, 0)


def run_chunks(c, layer, q, rows, seqs, starts, scale, window=0, ws=None, stream=None, q_pad=0, out_pad=0, fill=7.0, repeat=1):
    """The call's rows [tokens, heads, hd] as float64; q holds values of the type."""
    from gsdlq import hip
    if c.few_rows:
        seqs, starts = few(c, q, seqs, starts)
    n, (tokens, heads, hd) = len(starts) - 1, q.shape
    w = heads * hd
    qs = np.zeros((tokens, w + q_pad), np.float32)
    qs[:, :w] = q.reshape(tokens, w)
    one = row_bits(np.float32(fill), rows)
    dq, out = D(row_bits(qs, rows)), D(np.full((tokens, w + out_pad), one, one.dtype))
    ds, dt, ws = None if seqs is None else D(np.asarray(seqs, np.int32)), D(np.asarray(starts, np.int32)), ws or space(c, n, tokens, heads)
    for _ in range(repeat):
        c.lib.gsdh_paged_chunk_attention(stream, c.at, layer, p(dq), hip.ROW_TYPES[rows], w + q_pad, p(ds), p(dt), n, tokens, heads, scale, window,
                                         p(out), w + out_pad, p(ws), ws.nbytes)
    if stream is not None:
        c.lib.gsdh_stream_sync(stream)
    r = row_values(H(out, one.dtype, tokens * (w + out_pad)).reshape(tokens, w + out_pad), rows)
    assert (r[:, w:] == fill).all()
    return r[:, :w].reshape(tokens, heads, hd)


def attend_chunks(c, layer, q, seqs, starts, scale, window=0):
    """float64 out [tokens, heads, hd] (rows that no chunk names: NaN), and of each row and head, what its
    error is bounded by: sum P |V| per dim, the largest |score|, the largest sum |q k|, positions, largest |V|."""
    tokens, heads, hd = q.shape
    out, mag, big = (np.full((tokens, heads, hd), x) for x in (np.nan, 0.0, 0.0))
    top, dot, seen = (np.zeros((tokens, heads)) for _ in range(3))
    g = heads // c.kv
    for i in range(len(starts) - 1):
        s = i if seqs is None else seqs[i]
        if s < 0:
            continue
        m = starts[i + 1] - starts[i]
        for j in range(m):
            t, pos = starts[i] + j, int(c.lens[s]) - m + j
            first = max(0, pos + 1 - window) if window else 0
            at = np.arange(first, pos + 1)
            k, v = (c.values(w, layer, s, at) for w in (0, 1))
            for h in range(heads):
                qh, kh, vh = q[t, h].astype(np.float64), k[:, h // g], v[:, h // g]
                x = kh @ qh * scale
                e = np.exp(x - x.max())
                e /= e.sum()
                out[t, h], mag[t, h], big[t, h] = e @ vh, e @ np.abs(vh), np.abs(vh).max()
                top[t, h], dot[t, h], seen[t, h] = np.abs(x).max(), (np.abs(kh) @ np.abs(qh)).max() * abs(scale), len(at)
    return out, mag, top, dot, seen, big


def check(got, want, rows, exact_dots=False):
    """Within the rounding of the operator, derived in the test files that call it."""
    want, mag, top, dot, seen, big = want
    named = ~np.isnan(want).all(-1)
    assert (got[~named.any(-1)] == 7.0).all()   # rows that no chunk names
    eps = 2 * ((0 if exact_dots else got.shape[2] + 16) * dot + 8 * top) + seen * 5 / 8 + 160
    # The weights' fp16 parts are of 2^14 times the weight: half of fp16's least number, 2^-25, is 2^-39 of the
    # largest weight (which is 1, and so the sum is at least 1); each weight may lose that in either part
    bound = STEP * eps[..., None] * mag + seen[..., None] * big * 2.0 ** -38 + 1e-30
    if rows != "f32":
        # (an output below fp16's normal range: half of its least number, 2^-24)
        bound += HALF[rows] * (mag + np.abs(want)) * 1.01 + (2.0 ** -25 if rows == "f16" else 0)
    assert np.isfinite(got[named]).all()
    off = (np.abs(got - want) / bound)[named]
    assert off.size == 0 or off.max() <= 1, (off.max(), np.argwhere((np.abs(got - want) > bound) & named[..., None])[:3].tolist())


def chunk_cache(kind, lens, page, kv, hd, head_major, rng, values, layers=1, spare=5, few_rows=False):
    """few_rows: its calls go by few rows, else by many where the tables hold less than 1024 positions."""
    need, width = sum(-(-n // page) for n in lens), max(lens) // page + 2
    c = Cache(kind, layers, need + spare, page, kv, hd, head_major, len(lens), max(width, -(-FEW_ROOM // page)) if few_rows else width)
    c.few_rows = few_rows
    return c.fill(lens, rng, values)
