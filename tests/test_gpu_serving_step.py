"""A step of a serving loop from the operators it is made of, captured once and
replayed for other mixes of prompts, single tokens and padding: pages taken, rows
rotated and appended, chunks attended, logits adjusted, the next tokens and
their log probabilities.  Each stage against its definition over what the stage
before it left on the device."""
import ctypes

import numpy as np
import pytest

from chunk_util import attend_chunks, check as check_rows
from gpu_util import D, H, banner, p
from paged_util import Cache, decode, grid, ints, normal
from test_gpu_logit_rules import adjusted, check as check_logits, make
from test_gpu_rope import KV_HALF, LEAST, TURN, frequencies, rope, turn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()
    return hip.lib()


@pytest.mark.parametrize("kind,width", [("f16", 16), ("e4m3", 130)])
def test_step(lib, kind, width):
    """width 16: calls by many rows, 130 (of 8 positions): by few."""
    from gsdlq import hip
    banner(f"serving step {kind}, tables of {width}")
    rng = np.random.default_rng(width)
    heads, kv, hd, rd, page, n_seqs, chunks, tokens, vocab, scale = 8, 2, 64, 32, 8, 6, 5, 40, 3000, 0.125
    c = Cache(kind, 2, 200, page, kv, hd, False, n_seqs, width).fill([7, 8, 30, 0, 0, 1], rng, grid)
    c.few_rows = False
    w = (heads + 2 * kv) * hd
    d_freqs, r = rope(frequencies(lib, rd, "by_parts", 4.0), 0, 1.1)
    freqs = frequencies(lib, rd, "by_parts", 4.0)
    rules = make(rng, chunks, vocab, 30, 6, 3)
    keep = {k: D(v) for k, v in rules.items()}
    lr = hip.GsdLogitRules(history_width=30, n_bias=len(rules["bias_ids"]), n_masks=3, mask_words=rules["masks"].shape[1],
                           **{k: d.ptr for k, d in keep.items()})
    zeros = lambda *s: D(np.zeros(s, np.float32))  # noqa: E731
    dx, dq, out, logits = zeros(tokens, w), zeros(tokens, heads * hd), zeros(tokens, heads * hd), zeros(chunks, vocab)
    every, counts, seqs, starts = ints(range(n_seqs)), ints([0] * n_seqs), ints([-1] * chunks), ints([0] * (chunks + 1))
    rows, pos = ints([-1] * tokens), ints([0] * tokens)
    chosen, lp, en = ints([0] * chunks), zeros(chunks), zeros(chunks)
    ids, tops = ints([0] * chunks), zeros(chunks)
    need = lib.gsdh_token_logprobs_workspace_bytes(chunks, vocab, 1)
    lws = D(np.zeros(max(need, 16), np.uint8))
    aws = D(np.zeros(lib.gsdh_paged_chunk_attention_workspace_bytes(c.at, chunks, tokens, heads), np.uint8))
    at = lambda h: ctypes.c_void_p(dx.ptr.value + 4 * h * hd)  # noqa: E731
    st, ge = ctypes.c_void_p(), ctypes.c_void_p()
    lib.gsdh_stream_create(ctypes.byref(st))
    lib.gsdh_stream_begin_capture(st)
    lib.gsdh_pages_take(st, c.at, p(every), p(counts), n_seqs)
    lib.gsdh_paged_rope_append(st, c.at, 1, ctypes.byref(r), 0, at(0), w, at(heads), w, at(heads + kv), w, p(dq), heads * hd, p(rows), p(pos),
                               tokens, heads)
    lib.gsdh_paged_chunk_attention(st, c.at, 1, p(dq), 0, heads * hd, p(seqs), p(starts), chunks, tokens, heads, scale, 0, p(out), heads * hd,
                                   p(aws), aws.nbytes)
    lib.gsdh_logits_adjust(st, ctypes.byref(lr), p(logits), 0, vocab, chunks, vocab, p(logits), vocab)
    lib.gsdh_token_logprobs(st, p(logits), 0, vocab, chunks, vocab, p(chosen), 1, p(lp), p(en), p(ids), p(tops), p(lws), need)
    lib.gsdh_stream_end_capture(st, ctypes.byref(ge))

    def put(buf, a, dtype):
        a = np.ascontiguousarray(a, dtype)
        lib.gsdh_memcpy_h2d(buf.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes, None)
        lib.gsdh_stream_sync(None)

    for step in ({3: 20, 0: 1, 2: 1}, {0: 1, 1: 1, 2: 1, 3: 1, 4: 17}, {5: 33}, {}, {4: 3, 3: 1, 0: 2, 1: 30}):
        order = list(step)
        new = [step[s] for s in order]
        first = np.cumsum([0] + new).tolist()
        where = [int(c.lens[s]) + j for s in order for j in range(step[s])]
        whose = [s for s in order for _ in range(step[s])]
        x, y = normal(rng, (tokens, heads + 2 * kv, hd)), 3 * normal(rng, (chunks, vocab))
        put(counts, [step.get(s, 0) for s in range(n_seqs)], np.int32)
        put(seqs, order + [-1] * (chunks - len(order)), np.int32)
        put(starts, first + [first[-1]] * (chunks - len(order)), np.int32)
        put(rows, whose + [-1] * (tokens - len(whose)), np.int32)
        put(pos, where + [0] * (tokens - len(where)), np.int32)
        put(dx, x.reshape(tokens, w), np.float32)
        put(out, np.full((tokens, heads * hd), 7), np.float32)
        put(logits, y, np.float32)
        token = rng.integers(0, vocab, chunks)
        put(chosen, token, np.int32)
        lib.gsdh_graph_replay(ge, st)
        lib.gsdh_stream_sync(st)
        # what the page operators and the append left is the model from here on
        c.lens, c.tables, c.refs = c.download("lens"), c.download("tables"), c.download("refs")
        c.k, c.v = c.download("k"), c.download("v")
        n = len(whose)
        assert c.status() == 0
        if n:
            want, mag = turn(x[:n, heads:heads + kv], freqs, where, 0, 1.1)
            for t in range(n):
                for which, (row, m) in enumerate(((want[t], mag[t]), (x[t, heads + kv:].astype(np.float64), 0 * mag[t]))):
                    got = c.values(which, 1, whose[t], [where[t]])[0]
                    s = 1.0 if c.scales is None else c.scales[which, 1].astype(np.float64)[:, None]
                    off = np.abs(got - row)
                    assert (off <= TURN * m + KV_HALF[kind] * (np.abs(row) + TURN * m) + LEAST[kind] * s + 2.0 ** -23 * np.abs(row)).all()
        q = H(dq, np.float32, tokens * heads * hd).reshape(tokens, heads, hd)
        got = H(out, np.float32, tokens * heads * hd).reshape(tokens, heads, hd).astype(np.float64)
        check_rows(got, attend_chunks(c, 1, q, order, first, np.float32(scale)), "f32")
        z = H(logits, np.float32, chunks * vocab).reshape(chunks, vocab).astype(np.float64)
        want, mag = adjusted(y, rules)
        check_logits(z, want, mag, "f32")
        best, got = H(ids, np.int32, chunks), H(lp, np.float32, chunks)
        for i in range(chunks):
            if np.isneginf(z[i]).all():
                assert np.isnan(got[i])
                continue
            assert best[i] == z[i].argmax()
            ln = z[i, token[i]] - (z[i].max() + np.log(np.exp(z[i] - z[i].max()).sum()))
            assert got[i] == ln if np.isneginf(ln) else abs(got[i] - ln) < 1e-4
    lib.gsdh_graph_destroy(ge)
    lib.gsdh_stream_destroy(st)
