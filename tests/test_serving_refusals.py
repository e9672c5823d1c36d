"""What chunk attention's, the rotation's and the logit rules' entry points refuse:
every check is the host's, made before anything is launched, so it needs no GPU.
And the frequencies, which are the host's too."""
import ctypes
import math

import numpy as np
import pytest

from gsdlq import build, hip
from test_paged_refusals import BAD_CACHES, BUF, cache

pytestmark = pytest.mark.skipif(not __import__("os").path.exists(build.HIP_LIB), reason="engine library not built")


@pytest.fixture(scope="module")
def lib():
    return hip.lib()


def chunks(lib, c=None, layer=0, q=BUF, dtype=0, q_stride=256, seqs=BUF, starts=BUF, n=4, tokens=50, heads=4, scale=0.1, window=0, out=BUF,
           out_stride=256, ws=BUF, ws_bytes=1 << 40):
    lib.gsdh_paged_chunk_attention(None, ctypes.byref(c or cache()), layer, q, dtype, q_stride, seqs, starts, n, tokens, heads, scale, window, out,
                                   out_stride, ws, ws_bytes)


def rope(**other):
    f = dict(freqs=BUF, rotary_dim=64, interleaved=0, scale=1.0)
    f.update(other)
    return hip.GsdRope(**f)


def rows(lib, r=None, x=BUF, dtype=0, xs=256, out=BUF + 65536, os_=256, pos=BUF, n=3, heads=4, hd=64):
    r = r or rope()
    lib.gsdh_rope_rows(None, ctypes.byref(r), x, dtype, xs, out, os_, pos, n, heads, hd)


def append(lib, c=None, layer=0, r=None, dtype=0, q=BUF, qs=256, k=BUF, ks=128, v=BUF, vs=128, o=BUF + 4096, os_=256, seqs=BUF, pos=BUF, n=3, heads=4):
    r = r or rope()
    lib.gsdh_paged_rope_append(None, ctypes.byref(c or cache()), layer, ctypes.byref(r), dtype, q, qs, k, ks, v, vs, o, os_, seqs, pos, n, heads)


def adjust(lib, x=BUF, dtype=0, xs=100, n=2, vocab=100, out=BUF + 65536, os_=100, **rules):
    r = hip.GsdLogitRules(**rules)
    lib.gsdh_logits_adjust(None, ctypes.byref(r), x, dtype, xs, n, vocab, out, os_)


@pytest.mark.parametrize("other,text", BAD_CACHES)
def test_caches(lib, other, text):
    c = cache(**other)
    for call in (lambda: chunks(lib, c), lambda: append(lib, c)):
        with pytest.raises(hip.HipError, match=text):
            call()
    assert lib.gsdh_paged_chunk_attention_workspace_bytes(ctypes.byref(c), 1, 1, 4) == 0


@pytest.mark.parametrize("other,text", [
    (dict(layer=2), "layer 2"), (dict(layer=-1), "layer -1"), (dict(dtype=3), "type 3"), (dict(dtype=-1), "type -1"), (dict(dtype=2), "cache's type"),
    (dict(heads=3), "3 heads"), (dict(heads=34, q_stride=4096, out_stride=4096), "34 heads"), (dict(heads=0), "0 heads"), (dict(n=-1), "-1 chunks"),
    (dict(tokens=-1), "-1 tokens"), (dict(tokens=(1 << 30) + 1), "1073741825 tokens"), (dict(n=(1 << 20) + 1), "1048577 chunks"), (dict(seqs=None, n=5), "5 chunks, 4 sequences"), (dict(window=-1), "window -1"), (dict(q=None), "rows of q"),
    (dict(q=BUF + 4), "rows of q"), (dict(q_stride=258), "rows of q"), (dict(q_stride=-256), "rows of q"), (dict(out=BUF + 8), "rows of q"),
    (dict(out_stride=252), "at least 256"), (dict(dtype=1, q_stride=260), "rows of q"), (dict(starts=None), "null starts"),
    (dict(ws=None), "0 bytes of workspace"), (dict(ws_bytes=100), "100 bytes of workspace"), (dict(ws=BUF + 8), "not 16-byte aligned")])
def test_chunks(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        chunks(lib, **other)


def test_rows_of_16_bits_over_caches(lib):
    for kind, dtype in ((0, 2), (1, 1)):
        with pytest.raises(hip.HipError, match="cache's type"):
            chunks(lib, cache(dtype=kind), dtype=dtype)


def test_chunk_workspace(lib):
    """More tokens never need less; an invalid shape has none."""
    for c in (cache(), cache(head_dim=256, n_kv_heads=7), cache(head_dim=128, n_kv_heads=1024)):
        heads = c.n_kv_heads * 2
        sizes = [lib.gsdh_paged_chunk_attention_workspace_bytes(ctypes.byref(c), 4, t, heads) for t in (0, 1, 2, 7, 16, 64, 65, 1000, 1 << 20)]
        assert sizes == sorted(sizes) and sizes[1] > 0
        need = lib.gsdh_paged_chunk_attention_workspace_bytes(ctypes.byref(c), 4, 50, heads)
        w = heads * c.head_dim
        with pytest.raises(hip.HipError, match="bytes of workspace"):
            chunks(lib, c, heads=heads, q_stride=w, out_stride=w, ws_bytes=need - 1)
    for bad in ((-1, 5, 4), (1, -1, 4), (1, 5, 3), (1, 5, 0), (1, 5, 34)):
        assert lib.gsdh_paged_chunk_attention_workspace_bytes(ctypes.byref(cache()), *bad) == 0
    assert lib.gsdh_paged_chunk_attention_workspace_bytes(None, 1, 1, 4) == 0


@pytest.mark.parametrize("other,text", [
    (dict(r=rope(rotary_dim=0)), "rotary_dim 0"), (dict(r=rope(rotary_dim=7)), "rotary_dim 7"), (dict(r=rope(rotary_dim=66)), "rotary_dim 66"),
    (dict(r=rope(freqs=None)), "frequencies"), (dict(r=rope(freqs=BUF + 4)), "frequencies"), (dict(dtype=3), "type 3"), (dict(n=-1), "-1 tokens"),
    (dict(n=(1 << 30) + 1), "1073741825 tokens"), (dict(heads=0), "0 heads"), (dict(heads=16385), "16385 heads")])
def test_rotations(lib, other, text):
    for call in (rows, append):
        with pytest.raises(hip.HipError, match=text):
            call(lib, **other)


@pytest.mark.parametrize("other,text", [
    (dict(hd=4), "head_dim 4"), (dict(hd=68), "head_dim 68"), (dict(hd=1032), "head_dim 1032"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(pos=None), "null"), (dict(x=BUF + 8), "alignment"), (dict(xs=258), "whole 16 bytes"), (dict(dtype=1, xs=260), "whole 16 bytes"),
    (dict(xs=-256), "whole 16 bytes"), (dict(os_=252), "at least 256"), (dict(out=BUF, os_=512), "in place"), (dict(out=BUF, xs=0, os_=256), "at least 256")])
def test_rope_rows(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        rows(lib, **other)


@pytest.mark.parametrize("other,text", [
    (dict(layer=2), "layer 2"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(seqs=None), "null"), (dict(pos=None), "null"),
    (dict(q=BUF + 4), "alignment"), (dict(ks=130), "whole 16 bytes"), (dict(vs=-4), "whole 16 bytes"), (dict(os_=128), "at least 256"),
    (dict(o=BUF, os_=512), "in place"), (dict(dtype=2, ks=132), "whole 16 bytes")])
def test_append(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        append(lib, **other)


B = BUF
@pytest.mark.parametrize("other,text", [
    (dict(dtype=3), "type 3"), (dict(n=-1), "-1 rows"), (dict(vocab=0), "0 logits"), (dict(vocab=(1 << 24) + 1, xs=1 << 25, os_=1 << 25), "at most"),
    (dict(os_=99), "99 apart"), (dict(xs=-1), "apart"), (dict(out=BUF, xs=104, os_=108), "apart"), (dict(x=None), "null"), (dict(x=BUF + 2), "not aligned"),
    (dict(dtype=1, out=BUF + 65537), "not aligned"), (dict(history=B, history_width=4), "lengths"), (dict(history=B, history_lens=B, history_width=-1), "width"),
    (dict(history=B, history_lens=B, history_width=(1 << 30) + 1), "1073741825 tokens"), (dict(bias_starts=B, bias_ids=B, bias=B, n_bias=(1 << 30) + 1), "1073741825 biases"),
    (dict(repetition=B), "need a history"), (dict(presence=B), "need a history"), (dict(bias_starts=B, bias_ids=B), "go together"),
    (dict(bias_starts=B, bias=B), "go together"), (dict(bias=B), "go together"), (dict(bias_ids=B), "go together"),
    (dict(bias_starts=B, bias_ids=B, bias=B, n_bias=-1), "go together"), (dict(masks=B, mask_words=4, n_masks=1), "mask_rows"),
    (dict(masks=B, mask_rows=B, mask_words=3, n_masks=1), "100 logits, have 3"), (dict(mask_rows=B), "mask_rows"),
    (dict(masks=B, mask_rows=B, mask_words=4, n_masks=-1), "mask_rows")])
def test_logit_rules(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        adjust(lib, **other)


def test_null_structs(lib):
    with pytest.raises(hip.HipError, match="null rules"):
        lib.gsdh_logits_adjust(None, None, BUF, 0, 100, 1, 100, BUF, 100)
    with pytest.raises(hip.HipError, match="null rope"):
        lib.gsdh_rope_rows(None, None, BUF, 0, 64, BUF, 64, BUF, 1, 1, 64)
    with pytest.raises(hip.HipError, match="null cache"):
        lib.gsdh_paged_chunk_attention(None, None, 0, BUF, 0, 64, BUF, BUF, 1, 1, 1, 1.0, 0, BUF, 64, BUF, 1 << 40)


def test_nothing_to_do(lib):
    """Empty calls pass without a device."""
    chunks(lib, n=0)
    chunks(lib, tokens=0)
    rows(lib, n=0)
    append(lib, n=0)
    adjust(lib, n=0)


def frequencies(lib, kind, theta=1e6, rd=64, factor=1.0, context=8192.0, low=1.0, high=4.0):
    f = np.empty(max(rd // 2, 1))
    lib.gsdh_rope_frequencies(kind if isinstance(kind, int) else hip.ROPE_KINDS[kind], theta, rd, factor, context, low, high, hip.ptr(f))
    return f


@pytest.mark.parametrize("rd", [2, 20, 64, 128])
def test_frequencies(lib, rd):
    i = np.arange(rd // 2)
    plain = 1e6 ** (-2.0 * i / rd)
    near = lambda a, b: np.abs(a / b - 1).max() < 1e-13  # noqa: E731
    assert near(frequencies(lib, "plain", rd=rd), plain)
    assert near(frequencies(lib, "linear", rd=rd, factor=4.0), plain / 4)
    if rd > 2:
        ntk = frequencies(lib, "ntk", rd=rd, factor=4.0)
        assert near(ntk, (1e6 * 4.0 ** (rd / (rd - 2))) ** (-2.0 * i / rd)) and ntk[0] == 1 and abs(ntk[-1] * 4 / plain[-1] - 1) < 1e-12
    turns = 8192 * plain / (2 * math.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    assert near(frequencies(lib, "by_parts", rd=rd, factor=8.0), keep * plain + (1 - keep) * plain / 8)


@pytest.mark.parametrize("kind,other,text", [
    (4, {}, "kind 4"), (-1, {}, "kind -1"), ("plain", dict(rd=0), "rotary_dim 0"), ("plain", dict(rd=5), "rotary_dim 5"), ("plain", dict(theta=0.0), "theta"),
    ("plain", dict(theta=float("nan")), "theta"), ("plain", dict(theta=float("inf")), "theta"), ("linear", dict(factor=0.0), "factor"),
    ("ntk", dict(factor=float("nan")), "factor"), ("ntk", dict(rd=2), "one pair"), ("by_parts", dict(context=0.0), "context"),
    ("by_parts", dict(low=4.0, high=4.0), "turns"), ("by_parts", dict(low=float("nan")), "turns")])
def test_frequency_refusals(lib, kind, other, text):
    with pytest.raises(hip.HipError, match=text):
        frequencies(lib, kind, **other)
    with pytest.raises(hip.HipError, match="null"):
        lib.gsdh_rope_frequencies(0, 1e6, 64, 1.0, 1.0, 1.0, 2.0, None)
