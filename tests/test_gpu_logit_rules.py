"""gsdh_logits_adjust against its definition in 64 bits.

Tolerances: a quotient or product, a product and two differences, a sum: each is off
by half a step of fp32 of what it forms, so the result by less than 2^-22 of |x| r +
frequency count + presence + |bias|; then half a step of the logits' type."""
import ctypes

import numpy as np
import pytest

from chunk_util import HALF, row_bits, row_values, rounded
from gpu_util import D, H, banner, p

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from gsdlq import hip
    hip.device_info()
    return hip.lib()


def make(rng, n, vocab, history=50, bias=5, masks=3, words=None):
    """Lists with repeats and with tokens outside the vocabulary."""
    words = words or -(-vocab // 32)
    some = rng.integers(0, vocab, (n, 20))
    hist = np.take_along_axis(some, rng.integers(0, 20, (n, max(history, 1))), 1).astype(np.int32)
    hist[rng.random(hist.shape) < 0.05] = -1
    hist[rng.random(hist.shape) < 0.05] = vocab
    lens = np.array([history if i % 3 == 0 else rng.integers(0, history + 1) for i in range(n)], np.int32)
    per = [bias if i % 2 == 0 else int(rng.integers(0, bias + 1)) for i in range(n)]
    ids = rng.integers(-1, vocab + 1, max(sum(per), 1)).astype(np.int32)
    if sum(per) > 3:
        ids[1] = ids[0]     # the same token twice in a row's list
    f = lambda lo, hi: rng.uniform(lo, hi, n).astype(np.float32)  # noqa: E731
    m = rng.integers(0, 2 ** 32, (max(masks, 1), words), dtype=np.uint64).astype(np.uint32)
    if masks > 1:
        m[1] = 0            # allows nothing
    if masks > 2:
        m[2] = 0xFFFFFFFF
    return dict(history=hist, history_lens=lens, prompt_lens=(lens // 2).astype(np.int32), repetition=f(0.7, 1.5), frequency=f(-0.3, 0.5),
                presence=f(-0.3, 0.5), bias_starts=np.cumsum([0] + per).astype(np.int32), bias_ids=ids,
                bias=rng.uniform(-4, 4, len(ids)).astype(np.float32), masks=m,
                mask_rows=np.array([i % (masks + 1) - 1 for i in range(n)], np.int32))


def adjusted(x, r):
    """float64 (rows, what the roundings add up to)."""
    n, vocab = x.shape
    y, mag = x.astype(np.float64).copy(), np.abs(x.astype(np.float64))
    for i in range(n):
        if r.get("history") is not None:
            h = r["history"][i, :r["history_lens"][i]]
            prompt = r["prompt_lens"][i] if r.get("prompt_lens") is not None else 0
            ok = lambda t: t[(t >= 0) & (t < vocab)]  # noqa: E731
            seen = np.unique(ok(h))
            if r.get("repetition") is not None:
                with np.errstate(invalid="ignore"):
                    rep = float(r["repetition"][i])
                    y[i, seen] = np.where(y[i, seen] > 0, y[i, seen] / rep, y[i, seen] * rep)
                mag[i, seen] *= max(rep, 1 / rep)
            said, count = np.unique(ok(h[prompt:]), return_counts=True)
            for name, times in (("frequency", count), ("presence", 1)):
                if r.get(name) is not None:
                    y[i, said] -= float(r[name][i]) * times
                    mag[i, said] += abs(float(r[name][i])) * times
        if r.get("bias_starts") is not None:
            a, b = r["bias_starts"][i:i + 2]
            for t, v in dict(zip(r["bias_ids"][a:b].tolist(), r["bias"][a:b].tolist())).items():
                if 0 <= t < vocab:
                    y[i, t] += v
                    mag[i, t] += abs(v)
        if r.get("masks") is not None and r["mask_rows"][i] >= 0:
            bits = np.unpackbits(r["masks"][r["mask_rows"][i]].view(np.uint8), bitorder="little")[:vocab]
            y[i, bits == 0] = -np.inf
    return y, mag


def run(lib, x, rows, r, pad=0, out_pad=0, in_place=False, shift=0, width=None):
    """The call's rows as float64; shift: elements that the buffers are off 16 bytes."""
    from gsdlq import hip
    n, vocab = x.shape
    keep = {k: D(v) for k, v in r.items() if v is not None}
    rules = hip.GsdLogitRules(**{k: d.ptr for k, d in keep.items()})
    if r.get("history") is not None:
        rules.history_width = r["history"].shape[1] if width is None else width
    if r.get("bias_ids") is not None:
        rules.n_bias = len(r["bias_ids"])
    if r.get("masks") is not None:
        rules.n_masks, rules.mask_words = r["masks"].shape
    src = np.full((n, vocab + pad), 9.0, np.float32)
    src[:, :vocab] = x
    bits = row_bits(src, rows).reshape(-1)
    es = bits.dtype.itemsize
    off = np.zeros(shift, bits.dtype)
    dx = D(np.concatenate([off, bits]))
    stride = vocab + (pad if in_place else out_pad)
    do = dx if in_place else D(np.concatenate([off, np.full(n * stride, row_bits(np.float32(9), rows))]))
    at = lambda d: ctypes.c_void_p(d.ptr.value + es * shift)  # noqa: E731
    lib.gsdh_logits_adjust(None, ctypes.byref(rules), at(dx), hip.LOGIT_TYPES[rows], vocab + pad, n, vocab, at(do), stride)
    out = row_values(H(do, bits.dtype, shift + n * stride)[shift:].reshape(n, stride), rows)
    assert (out[:, vocab:] == 9).all()
    return out[:, :vocab]


def check(got, want, mag, rows):
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine]) - (2.0 ** -22 * mag[fine] + HALF[rows] * (np.abs(want[fine]) + 2.0 ** -22 * mag[fine]) +
                                            (2.0 ** -25 if rows == "f16" else 0))
    assert np.isfinite(got[fine]).all() and (off.size == 0 or off.max() <= 0), off.max()


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab,pad,out_pad,shift", [(1, 1, 0, 0, 0), (5, 31, 1, 0, 0), (7, 4096, 0, 8, 0), (4, 4097, 3, 1, 1), (9, 12345, 0, 0, 3),
                                                       (3, 32768, 0, 0, 0), (2, 130001, 7, 7, 0)])
def test_everything_at_once(lib, rows, n, vocab, pad, out_pad, shift):
    """Every part, odd sizes and strides, buffers at any element; in place the same bits."""
    banner(f"logit rules {rows} {n} x {vocab}")
    rng = np.random.default_rng(vocab)
    x = rounded(3 * rng.standard_normal((n, vocab)), rows).astype(np.float32)
    x[rng.random(x.shape) < 0.02] = -np.inf
    for history, bias, masks in ((50, 5, 3), (3000, 400, 5), (0, 0, 1)):
        r = make(rng, n, vocab, history, bias, masks)
        got = run(lib, x, rows, r, pad, out_pad, shift=shift)
        check(got, *adjusted(x, r), rows)
        assert np.array_equal(got, run(lib, x, rows, r, pad, in_place=True, shift=shift))


@pytest.mark.parametrize("part", ["repetition", "frequency", "presence", "bias", "masks", "none"])
def test_each_part_alone(lib, part):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    r = make(rng, 6, 5000, 300, 20, 3, words=200)
    names = {"bias": ("bias_starts", "bias_ids", "bias"), "masks": ("masks", "mask_rows"), "none": ()}.get(part, (part, "history", "history_lens"))
    r = {k: v for k, v in r.items() if k in names}
    got = run(lib, x, "f32", r)
    check(got, *adjusted(x, r), "f32")
    assert np.array_equal(got, run(lib, x, "f32", r, in_place=True))
    if part == "none":
        assert np.array_equal(got, x)


def test_what_is_not_a_number(lib):
    """Forbidden logits are -inf whatever they were; others keep a NaN or an infinity; a mask that leaves nothing."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 100)).astype(np.float32)
    x[:, 3], x[:, 4], x[:, 5], x[:, 6] = np.nan, np.inf, -np.inf, np.inf
    masks = np.zeros((2, 4), np.uint32)
    masks[0, 0] = 0xFFFFFFBF     # not token 6
    r = dict(masks=masks, mask_rows=np.array([0, 1], np.int32), history=np.array([[4, 5], [4, 5]], np.int32),
             history_lens=np.array([2, 2], np.int32), repetition=np.array([1.5, 1.5], np.float32), frequency=np.array([1, 1], np.float32))
    for in_place in (False, True):
        got = run(lib, x, "f32", r, in_place=in_place)
        assert np.isnan(got[0, 3]) and got[0, 4] == np.inf and got[0, 5] == -np.inf and got[0, 6] == -np.inf
        assert np.array_equal(got[0, 7:32], x[0, 7:32]) and np.isneginf(got[0, 32:]).all() and np.isneginf(got[1]).all()


def test_counts(lib):
    """Counts far above one, the prompt's tokens apart from the answer's, the last of a token's biases."""
    x = np.full((2, 64), 2.0, np.float32)
    hist = np.zeros((2, 70000), np.int32)
    hist[:, 30:60] = 5
    hist[:, 60:] = 7
    r = dict(history=hist, history_lens=np.array([70000, 59], np.int32), prompt_lens=np.array([31, 60], np.int32),
             repetition=np.full(2, 2.0, np.float32), frequency=np.full(2, 2.0 ** -10, np.float32), presence=np.full(2, 0.5, np.float32),
             bias_starts=np.array([0, 4, 4], np.int32), bias_ids=np.array([9, 8, 9, 9], np.int32), bias=np.array([1, 2, 4, -8], np.float32))
    got = run(lib, x, "f32", r)
    want = np.full((2, 64), 2.0)
    want[:, [0, 5]] = 1.0
    want[0, 7] = 1.0 - 69940 * 2.0 ** -10 - 0.5
    want[0, 5] = 1.0 - 29 * 2.0 ** -10 - 0.5
    want[0, 8], want[0, 9] = 4.0, -6.0
    assert np.array_equal(got, want)


def test_rows_with_bad_lists_become_nan(lib):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((8, 300)).astype(np.float32)
    r = make(rng, 8, 300, 40, 6, 3)
    r["history_lens"][0], r["history_lens"][1] = -1, 41
    r["mask_rows"][2], r["mask_rows"][3] = 3, -2
    starts = r["bias_starts"].copy()
    starts[6] = starts[5] - 1 if starts[5] > 0 else -1      # row 5 falls; row 6 reads from there
    r["bias_starts"] = starts
    got = run(lib, x, "f32", r)
    assert np.isnan(got[[0, 1, 2, 3, 5]]).all()
    good = {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in r.items()}
    want, mag = adjusted(x[[4, 7]], {k: (v[[4, 7]] if k not in ("bias_starts", "bias_ids", "bias", "masks") else v) for k, v in good.items()} |
                         {"bias_starts": None})
    part = run(lib, x[[4, 7]], "f32", {k: (v[[4, 7]] if k not in ("bias_starts", "bias_ids", "bias", "masks") else v) for k, v in good.items()} |
               {"bias_starts": None, "bias_ids": None, "bias": None})
    check(part, want, mag, "f32")
    r["bias_starts"] = starts.copy()
    r["bias_starts"][8] = len(r["bias_ids"]) + 1
    assert np.isnan(run(lib, x, "f32", r)[7]).all()


def test_then_log_probabilities(lib):
    """The adjusted rows through the log probabilities: what is forbidden has probability 0, a row that has nothing is NaN."""
    from gsdlq import hip
    rng = np.random.default_rng(8)
    n, vocab = 6, 3001
    x = 3 * rng.standard_normal((n, vocab)).astype(np.float32)
    r = make(rng, n, vocab, 100, 10, 2)
    y, _ = adjusted(x, r)
    keep = {k: D(v) for k, v in r.items()}
    rules = hip.GsdLogitRules(history_width=100, n_bias=len(r["bias_ids"]), n_masks=2, mask_words=r["masks"].shape[1],
                              **{k: d.ptr for k, d in keep.items()})
    dx, tok = D(x), D(rng.integers(0, vocab, n).astype(np.int32))
    lib.gsdh_logits_adjust(None, ctypes.byref(rules), p(dx), 0, vocab, n, vocab, p(dx), vocab)
    need = lib.gsdh_token_logprobs_workspace_bytes(n, vocab, 3)
    ws, lp, en, ids, tl = D(np.zeros(max(need, 16), np.uint8)), D(np.zeros(n, np.float32)), D(np.zeros(n, np.float32)), D(np.zeros((n, 3), np.int32)), \
        D(np.zeros((n, 3), np.float32))
    lib.gsdh_token_logprobs(None, p(dx), 0, vocab, n, vocab, p(tok), 3, p(lp), p(en), p(ids), p(tl), p(ws), need)
    lp, ids = H(lp, np.float32, n), H(ids, np.int32, 3 * n).reshape(n, 3)
    tok = H(tok, np.int32, n)
    for i in range(n):
        if r["mask_rows"][i] == 1:
            assert np.isnan(lp[i])
            continue
        top = y[i].max()
        z = top + np.log(np.exp(y[i] - top).sum())
        want = y[i, tok[i]] - z
        assert lp[i] == want if np.isneginf(want) else abs(lp[i] - want) < 1e-4
        assert y[i, ids[i, 0]] > top - 1e-5
