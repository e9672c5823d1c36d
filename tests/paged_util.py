"""A paged cache on the device and its plain model in numpy: the same pools,
tables and counts, with the operators' definitions in 64 bits."""
import ctypes

import numpy as np

from gpu_util import D, E, H, p


def _e4m3_table():
    t = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[b] = np.nan if (b & 127) == 127 else -v if b & 128 else v
    return t


E4M3 = _e4m3_table()


def encode(x, kind):
    """float -> the bits of the type, rounded to nearest even (e4m3: clamped to +-448)."""
    x = np.asarray(x, np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    if kind == "bf16":
        u = x.view(np.uint32)
        r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)
    pos = E4M3[:127]   # rising
    a = np.minimum(np.abs(x.astype(np.float64)), 448.0)
    hi = np.clip(np.searchsorted(pos, np.nan_to_num(a)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dh, dl = pos[hi] - a, a - pos[lo]
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(pos[hi] == a, hi, code)
    code = np.where(np.isnan(x), 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def decode(bits, kind):
    """The bits' values, float64."""
    if kind == "f16":
        return bits.view(np.float16).astype(np.float64)
    if kind == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3[bits]


def nan_bits(shape, kind):
    return np.full(shape, 127, np.uint8) if kind == "e4m3" else np.full(shape, 0x7FFF, np.uint16)


class Cache:
    """Pools [layers][pages]..., host mirrors `k` and `v` of their bits."""

    def __init__(self, kind="f16", layers=1, pages=16, page=16, kv=2, hd=64, head_major=False, seqs=4, width=None, scales=None,
                 refs=True):
        from gsdlq import hip
        self.lib, self.kind, self.layers, self.pages, self.page, self.kv, self.hd = hip.lib(), kind, layers, pages, page, kv, hd
        self.head_major, self.seqs, self.width = head_major, seqs, width or pages
        shape = (layers, pages, kv, page, hd) if head_major else (layers, pages, page, kv, hd)
        self.k, self.v = nan_bits(shape, kind), nan_bits(shape, kind)   # (what nobody wrote is NaN)
        self.refs = np.zeros(pages, np.int32)
        self.tables = np.full((seqs, self.width), -1, np.int32)
        self.lens = np.zeros(seqs, np.int32)
        if kind == "e4m3" and scales is None:
            scales = np.exp2(np.random.default_rng(pages).integers(-2, 3, (2, layers, kv))).astype(np.float32)
        self.scales = scales
        self.has_refs, self.dev = refs, {}
        self.upload()

    def upload(self):
        self.dev = {n: D(getattr(self, n)) for n in ("k", "v", "refs", "tables", "lens")}
        self.dev["status"] = D(np.zeros(1, np.uint32))
        if self.scales is not None:
            self.dev["ks"], self.dev["vs"] = D(self.scales[0]), D(self.scales[1])
        self.c = self.struct()
        self.at = ctypes.byref(self.c)

    def struct(self, **other):
        from gsdlq import hip
        d = self.dev
        f = dict(k=d["k"].ptr, v=d["v"].ptr, k_scale=d["ks"].ptr if "ks" in d else None,
                 v_scale=d["vs"].ptr if "vs" in d else None, refs=d["refs"].ptr if self.has_refs else None,
                 tables=d["tables"].ptr, lens=d["lens"].ptr, status=d["status"].ptr, n_layers=self.layers, n_pages=self.pages,
                 page_size=self.page, n_kv_heads=self.kv, head_dim=self.hd, dtype=hip.KV_TYPES[self.kind],
                 head_major=int(self.head_major), n_seqs=self.seqs, table_width=self.width)
        f.update(other)
        return hip.GsdPagedCache(**f)

    def download(self, name):
        a = getattr(self, name)
        return H(self.dev[name], a.dtype, a.size).reshape(a.shape)

    def status(self):
        return int(H(self.dev["status"], np.uint32, 1)[0])

    def clear_status(self):
        self.dev["status"] = D(np.zeros(1, np.uint32))
        self.c = self.struct()
        self.at = ctypes.byref(self.c)

    # -- the model -------------------------------------------------------
    def rows(self, pool, layer, pos, table):
        """View-free index of rows [kv, hd] of positions `pos` of a table row."""
        pos = np.asarray(pos)
        pg, slot = table[pos // self.page], pos % self.page
        return (layer, pg, slice(None), slot) if self.head_major else (layer, pg, slot)

    def values(self, which, layer, seq, pos):
        """float64 [positions, kv, hd]."""
        x = decode((self.k, self.v)[which][self.rows(None, layer, pos, self.tables[seq])], self.kind)
        return x if self.scales is None else x * self.scales[which, layer].astype(np.float64)[:, None]

    def set_values(self, which, layer, seq, pos, x):
        if self.scales is not None:
            x = np.asarray(x, np.float32) / self.scales[which, layer][:, None]
        (self.k, self.v)[which][self.rows(None, layer, pos, self.tables[seq])] = encode(x, self.kind)

    def fill(self, lens, rng, values):
        """Sequences of these lengths on scattered pages, rows of values(rng, shape)."""
        need = [-(-n // self.page) for n in lens]
        order = rng.permutation(self.pages)[:sum(need)]
        assert len(order) == sum(need)
        at = 0
        for s, (n, k) in enumerate(zip(lens, need)):
            self.lens[s], self.tables[s, :k] = n, order[at:at + k]
            self.refs[order[at:at + k]] = 1
            at += k
            for layer in range(self.layers):
                for which in (0, 1):
                    if n:
                        self.set_values(which, layer, s, np.arange(n), values(rng, (n, self.kv, self.hd)))
        self.upload()
        return self

    def attend(self, layer, q, seqs, scale, window=0):
        """float64 (out, sum P |V|, largest |score| + 1, largest sum |q k|) for rows q [n, heads, hd]; padding rows NaN."""
        n, heads, hd = q.shape
        out, mag = np.full((n, heads, hd), np.nan), np.zeros((n, heads, hd))
        top, dot = np.zeros((n, heads)), np.zeros((n, heads))
        g = heads // self.kv
        for i, s in enumerate(seqs):
            if s < 0:
                continue
            end = int(self.lens[s])
            first = max(0, end - window) if window else 0
            if end == 0:
                out[i] = 0
                continue
            k, v = (self.values(w, layer, s, np.arange(first, end)) for w in (0, 1))
            for h in range(heads):
                qh, kh, vh = q[i, h].astype(np.float64), k[:, h // g], v[:, h // g]
                x = kh @ qh * scale
                e = np.exp(x - x.max())
                e /= e.sum()
                out[i, h], mag[i, h] = e @ vh, e @ np.abs(vh)
                top[i, h], dot[i, h] = np.abs(x).max(), (np.abs(kh) @ np.abs(qh)).max() * abs(scale)
        return out, mag, top, dot

    # -- the calls -------------------------------------------------------
    def space(self, n, heads):
        return D(np.zeros(self.lib.gsdh_paged_attention_workspace_bytes(self.at, n, heads), np.uint8))

    def run_attend(self, layer, q, seqs, scale, window=0, ws=None, stream=None, q_pad=0, out_pad=0, fill=7.0, identity=False):
        n, heads, hd = q.shape
        w = heads * hd
        qs = np.zeros((n, w + q_pad), np.float32)
        qs[:, :w] = q.reshape(n, w)
        out = D(np.full((n, w + out_pad), fill, np.float32))
        dq, ds, ws = D(qs), D(np.asarray(seqs, np.int32)), ws or self.space(n, heads)
        self.lib.gsdh_paged_attention(stream, self.at, layer, p(dq), w + q_pad, None if identity else p(ds), n, heads, scale, window,
                                      p(out), w + out_pad, p(ws), ws.nbytes)
        if stream is not None:
            self.lib.gsdh_stream_sync(stream)
        r = H(out, np.float32, n * (w + out_pad)).reshape(n, w + out_pad)
        assert (r[:, w:] == fill).all()
        return r[:, :w].reshape(n, heads, hd)


def grid(rng, shape):
    """Values of few bits: their products and sums are exact in fp32, and all three cache types hold them."""
    return rng.integers(-8, 9, shape).astype(np.float32) / 4


def normal(rng, shape):
    return rng.standard_normal(shape).astype(np.float32)


def ints(x):
    return D(np.asarray(x, np.int32))


def angles(n, hd, theta=1e6):
    """(cos, sin) [n, hd / 2, 2] of float32 angles."""
    f = (1.0 / np.float32(theta) ** (np.arange(0, hd, 2, dtype=np.float32) / np.float32(hd))).astype(np.float32)
    a = np.arange(n, dtype=np.float32)[:, None] * f
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def rotate(x, a, interleaved):
    """float32 rotation, products and sums rounded one by one; x [n, heads, hd], a [n, hd / 2, 2]."""
    c, s = a[:, None, :, 0], a[:, None, :, 1]
    h = x.shape[-1] // 2
    u, w = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    y, z = u * c - w * s, u * s + w * c
    return np.stack([y, z], -1).reshape(x.shape) if interleaved else np.concatenate([y, z], -1)
