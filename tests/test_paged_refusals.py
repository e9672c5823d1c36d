"""What the paged cache's and the log probabilities' entry points refuse: every
check is the host's, made before anything is launched, so it needs no GPU."""
import ctypes

import pytest

from gsdlq import build, hip

pytestmark = pytest.mark.skipif(not __import__("os").path.exists(build.HIP_LIB), reason="engine library not built")
BUF = 0x10000   # an aligned address; nothing reads it


@pytest.fixture(scope="module")
def lib():
    return hip.lib()


def cache(**other):
    f = dict(k=BUF, v=BUF, k_scale=None, v_scale=None, refs=BUF, tables=BUF, lens=BUF, status=BUF, n_layers=2, n_pages=64, page_size=16,
             n_kv_heads=2, head_dim=64, dtype=0, head_major=0, n_seqs=4, table_width=8)
    f.update(other)
    return hip.GsdPagedCache(**f)


def attend(lib, c=None, layer=0, q=BUF, q_stride=256, seqs=BUF, n=4, heads=4, scale=0.1, window=0, out=BUF, out_stride=256, ws=BUF,
           ws_bytes=1 << 40):
    lib.gsdh_paged_attention(None, ctypes.byref(c or cache()), layer, q, q_stride, seqs, n, heads, scale, window, out, out_stride, ws, ws_bytes)


def store(lib, c=None, layer=0, q=BUF, qs=256, k=BUF, ks=128, v=BUF, vs=128, o=BUF + 4096, os_=256, seqs=BUF, pos=BUF, n=3, heads=4,
          angles=BUF, n_angles=10):
    lib.gsdh_paged_rope_store(None, ctypes.byref(c or cache()), layer, q, qs, k, ks, v, vs, o, os_, seqs, pos, n, heads, angles, n_angles, 1)


def logprobs(lib, x=BUF, dtype=0, stride=1000, n=4, vocab=1000, tokens=BUF, top=2, lp=BUF, en=BUF, ids=BUF, tl=BUF, ws=BUF, ws_bytes=1 << 40):
    lib.gsdh_token_logprobs(None, x, dtype, stride, n, vocab, tokens, top, lp, en, ids, tl, ws, ws_bytes)


BAD_CACHES = [(dict(dtype=3), "cache type"), (dict(dtype=-1), "cache type"), (dict(head_dim=96), "head_dim 96"),
              (dict(page_size=12), "page_size 12"), (dict(page_size=4), "page_size 4"), (dict(page_size=512), "page_size 512"),
              (dict(n_layers=0), "0 layers"), (dict(n_pages=0), "0 pages"), (dict(n_pages=(1 << 20) + 1), "at most 2\\^20"),
              (dict(n_kv_heads=0), "0 KV heads"), (dict(table_width=0), "tables of 0"), (dict(n_seqs=0), "n_seqs 0"),
              (dict(n_seqs=8193), "n_seqs 8193"), (dict(table_width=1 << 27), "tables of"), (dict(k=None), "null buffer"),
              (dict(tables=None), "null buffer"), (dict(lens=None), "null buffer"), (dict(status=None), "null buffer"),
              (dict(v=BUF + 8), "16-byte aligned"), (dict(dtype=2), "scales"), (dict(k_scale=BUF, v_scale=BUF), "scales"),
              (dict(dtype=2, k_scale=BUF), "scales")]


@pytest.mark.parametrize("other,text", BAD_CACHES)
def test_caches(lib, other, text):
    c = cache(**other)
    at = ctypes.byref(c)
    calls = [lambda: attend(lib, c), lambda: store(lib, c), lambda: lib.gsdh_pages_take(None, at, BUF, BUF, 1),
             lambda: lib.gsdh_pages_fork(None, at, BUF, BUF, 1, BUF, 1 << 40), lambda: lib.gsdh_pages_free(None, at, BUF, 1),
             lambda: lib.gsdh_pages_compact(None, at, None, BUF, 1 << 40), lambda: lib.gsdh_pages_copy(None, at, BUF, BUF, 1, BUF, 1 << 40)]
    for call in calls:
        with pytest.raises(hip.HipError, match=text):
            call()
    assert lib.gsdh_pages_workspace_bytes(at) == 0
    assert lib.gsdh_paged_attention_workspace_bytes(at, 1, 4) == 0


def test_positions_of_one_call(lib):
    c = cache(table_width=1 << 22, page_size=256, n_seqs=100)
    with pytest.raises(hip.HipError, match="100 rows of up to 1073741824 positions"):
        attend(lib, c, n=100)
    assert lib.gsdh_paged_attention_workspace_bytes(ctypes.byref(c), 100, 4) == 0
    assert lib.gsdh_paged_attention_workspace_bytes(ctypes.byref(c), 10, 4) > 0


def test_null_cache(lib):
    with pytest.raises(hip.HipError, match="null cache"):
        lib.gsdh_pages_free(None, None, BUF, 1)
    assert lib.gsdh_paged_attention_workspace_bytes(None, 1, 4) == 0


@pytest.mark.parametrize("other,text", [
    (dict(layer=2), "layer 2"), (dict(layer=-1), "layer -1"), (dict(heads=3), "3 heads"), (dict(heads=34, q_stride=4096, out_stride=4096), "34 heads"),
    (dict(heads=0), "0 heads"), (dict(n=-1), "-1 rows"), (dict(seqs=None, n=5), "5 rows, 4 sequences"), (dict(window=-1), "window -1"),
    (dict(q=None), "rows of q"), (dict(q=BUF + 4), "rows of q"), (dict(q_stride=258), "rows of q"), (dict(q_stride=-256), "rows of q"),
    (dict(out=BUF + 8), "rows of q"), (dict(out_stride=252), "at least 256"), (dict(ws=None), "0 bytes of workspace"),
    (dict(ws_bytes=100), "100 bytes of workspace"), (dict(ws=BUF + 8), "not 16-byte aligned")])
def test_attention(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        attend(lib, **other)


@pytest.mark.parametrize("other,text", [
    (dict(layer=2), "layer 2"), (dict(n=-1), "-1 tokens"), (dict(heads=0), "0 heads"), (dict(n_angles=-1), "angles of -1"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(seqs=None), "null"), (dict(pos=None), "null"), (dict(angles=None), "null"), (dict(q=BUF + 4), "alignment"),
    (dict(ks=130), "multiples of 4"), (dict(vs=-4), "multiples of 4"), (dict(os_=128), "at least 256"), (dict(angles=BUF + 8), "alignment"),
    (dict(o=BUF, os_=512), "in place")])
def test_store(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        store(lib, **other)


def test_pages(lib):
    c = cache()
    at = ctypes.byref(c)
    ws = lib.gsdh_pages_workspace_bytes(at)
    assert ws > 0
    for call in (lambda n, a=BUF, b=BUF: lib.gsdh_pages_take(None, at, a, b, n), lambda n, a=BUF, b=BUF: lib.gsdh_pages_fork(None, at, a, b, n, BUF, ws),
                 lambda n, a=BUF, b=BUF: lib.gsdh_pages_free(None, at, a if b else None, n)):
        for n in (-1, 5):
            with pytest.raises(hip.HipError, match="list of"):
                call(n)
        for a, b in ((None, BUF), (BUF, None)):
            with pytest.raises(hip.HipError, match="null list"):
                call(2, a, b)
    with pytest.raises(hip.HipError, match="list of 65"):
        lib.gsdh_pages_copy(None, at, BUF, BUF, 65, BUF, ws)
    for fn, args in (("gsdh_pages_fork", (BUF, BUF, 1)), ("gsdh_pages_copy", (BUF, BUF, 1)), ("gsdh_pages_compact", (None,))):
        with pytest.raises(hip.HipError, match="bytes of workspace"):
            getattr(lib, fn)(None, at, *args, BUF, ws - 1)
        with pytest.raises(hip.HipError, match="not 16-byte aligned"):
            getattr(lib, fn)(None, at, *args, BUF + 4, ws)
    none = cache(refs=None)
    for fn, args in (("gsdh_pages_take", (BUF, BUF, 1)), ("gsdh_pages_fork", (BUF, BUF, 1, BUF, ws)), ("gsdh_pages_free", (BUF, 1)),
                     ("gsdh_pages_compact", (None, BUF, ws))):
        with pytest.raises(hip.HipError, match="null buffer"):
            getattr(lib, fn)(None, ctypes.byref(none), *args)


@pytest.mark.parametrize("other,text", [
    (dict(dtype=3), "type 3"), (dict(n=-1), "-1 rows"), (dict(vocab=0), "0 logits"), (dict(vocab=1 << 20, stride=1 << 20), "at most"),
    (dict(top=33), "33 alternatives"), (dict(top=-1), "-1 alternatives"), (dict(vocab=1, top=2), "2 alternatives"), (dict(stride=999), "999 apart"),
    (dict(lp=None), "go together"), (dict(tokens=None), "go together"), (dict(ids=None), "no buffers"), (dict(tl=None), "no buffers"),
    (dict(x=None), "null"), (dict(x=BUF + 2), "not aligned"), (dict(x=BUF + 1, dtype=1), "not aligned"),
    (dict(vocab=9000, stride=9000, ws=None), "bytes of workspace"), (dict(vocab=9000, stride=9000, ws_bytes=64), "bytes of workspace"),
    (dict(vocab=9000, stride=9000, ws=BUF + 4), "not 16-byte")])
def test_logprobs(lib, other, text):
    with pytest.raises(hip.HipError, match=text):
        logprobs(lib, **other)


def test_nothing_to_do(lib):
    """Empty calls pass without a device."""
    attend(lib, n=0)
    store(lib, n=0)
    logprobs(lib, n=0)
    c = cache()
    lib.gsdh_pages_take(None, ctypes.byref(c), None, None, 0)
    lib.gsdh_pages_free(None, ctypes.byref(c), None, 0)


def test_workspace_sizes(lib):
    """More rows never need less; a call's own need is covered for fewer rows too."""
    for vocab in (300, 2041, 2048, 8185, 8186, 9000, 130001, (1 << 20) - 8):
        for top in (0, 1, 32):
            sizes = [lib.gsdh_token_logprobs_workspace_bytes(n, vocab, top) for n in range(1, 700)]
            assert sizes == sorted(sizes)
    c = cache()
    sizes = [lib.gsdh_paged_attention_workspace_bytes(ctypes.byref(c), n, 4) for n in (1, 2, 64, 1000, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
