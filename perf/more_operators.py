"""What the operators around a chunk of new tokens are measured on: attention of
several sequences' chunks over the paged cache, rotary positions (part of the
head, scaled contexts; rows to rows, and rows to the cache), and what is done to
logits before a token is chosen (penalties, biases, grammar masks), each through
the calls that a program makes (the C ABI of `gsdlq.hip`), beside their plain
forms in torch.

Head shapes are those of the benchmark and the tests, contexts go up to 32768
positions (131072 for positions alone), vocabularies to some 130,000 entries.
Lengths, pages, lists' lengths and positions come from the case alone, every
value from the seed.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

THETA = 1e6
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "e4m3": 1, "f32": 4}
HEADS = ((32, 8, 128), (32, 8, 128), (16, 4, 128), (16, 8, 64), (4, 2, 64), (8, 8, 128), (12, 4, 64), (16, 2, 256))
MOST_SCORES = 32 * 2048 * 32768   # heads * tokens * positions of the largest case


def listed():
    b = dict(heads=32, kv=8, hd=128, dtype="f16", rows="f32", page=16, order="slot")
    return [
        # a short question to the small test model, in one piece
        dict(b, name="chunk_short", kind="chunk", heads=4, kv=2, hd=64, batch=1, ctx=33, new=7, ragged=False, window=0),
        # five drafted tokens of each of sixteen users, to be verified over what they have said so far
        dict(b, name="chunk_drafts", kind="chunk", batch=16, ctx=8191, new=5, ragged=True, window=0),
        # a long prompt from its first token on
        dict(b, name="chunk_prompt", kind="chunk", batch=1, ctx=4096, new=4096, ragged=False, window=0),
        # the last piece of a document of 32768 positions, in 16 bits throughout
        dict(b, name="chunk_document", kind="chunk", dtype="bf16", rows="bf16", page=64, batch=1, ctx=32768, new=2048, ragged=False, window=0),
        # a served step: prompts of every length beside users who wait for one token, 8-bit cache, a sliding window
        dict(b, name="chunk_mixed_e4m3", kind="chunk", dtype="e4m3", order="head", page=32, batch=24, ctx=6001, new=700, ragged=True, window=4096),
        # q and K rows of a step of 64 users, slow frequencies stretched eightfold for a long context
        dict(name="rope_step", kind="rope", heads=40, hd=128, turned=128, rows="f32", tokens=64, far=131072, interleaved=1, factor=8.0),
        # a prompt's rows in 16 bits, half of each head turned
        dict(name="rope_prompt", kind="rope", heads=40, hd=128, turned=64, rows="bf16", tokens=8191, far=32768, interleaved=0, factor=1.0),
        # the rows of a decode step into the cache
        dict(b, name="append_step", kind="append", batch=64, tokens=64, ctx=3000, turned=128, interleaved=1, factor=4.0),
        # pieces of several prompts in one call, 16-bit rows into an 8-bit cache, a quarter of each head turned
        dict(b, name="append_prompts", kind="append", dtype="e4m3", rows="bf16", order="head", page=32, batch=5, tokens=4099, ctx=700, turned=32,
             interleaved=0, factor=1.0),
        # one user's next token: penalties over an answer so far, a few biases
        dict(name="logits_token", kind="logits", rows="f32", batch=1, vocab=32768, pad=0, history=900, bias=16, masks=0),
        # a batch whose answers have to keep to grammars
        dict(name="logits_batch", kind="logits", rows="f32", batch=256, vocab=32768, pad=0, history=2000, bias=300, masks=8),
        # a large odd vocabulary in 16 bits, long histories
        dict(name="logits_large", kind="logits", rows="bf16", batch=61, vocab=130001, pad=7, history=8000, bias=40, masks=3),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "chunk", "chunk", "rope", "append", "logits", "logits"))
    if kind == "logits":
        vocab = _log_int(rng, 257, 140000)
        return dict(kind=kind, rows=rng.choice(("f32", "f32", "bf16", "f16")), batch=_log_int(rng, 1, min(512, 8000000 // vocab)), vocab=vocab,
                    pad=rng.choice((0, 0, 1, 8)), history=rng.choice((0, _log_int(rng, 1, 8000))), bias=rng.choice((0, 3, 300)),
                    masks=rng.choice((0, 1, 5)))
    heads, kv, hd = rng.choice(HEADS)
    turned = rng.choice((hd, hd, hd // 2, hd // 4, 20))
    if kind == "rope":
        return dict(kind=kind, heads=heads + kv, hd=hd, turned=turned, rows=rng.choice(("f32", "bf16", "f16")),
                    tokens=_log_int(rng, 1, min(8191, 8191 * 5120 // ((heads + kv) * hd))), far=_log_int(rng, 100, 131072),
                    interleaved=rng.randrange(2), factor=rng.choice((1.0, 4.0, 8.0)))
    dtype = rng.choice(("f16", "f16", "bf16", "e4m3"))
    rows = rng.choice(("f32", dtype if dtype != "e4m3" else rng.choice(("f16", "bf16"))))
    c = dict(kind=kind, heads=heads, kv=kv, hd=hd, dtype=dtype, rows=rows, page=rng.choice((8, 16, 16, 32, 64, 128)),
             order=rng.choice(("slot", "slot", "head")))
    if kind == "chunk":
        batch = _log_int(rng, 1, 32)
        new = _log_int(rng, 1, 2048)
        most = min(32768, MOST_SCORES * 128 // (heads * hd * batch * new))
        return dict(c, batch=batch, ctx=_log_int(rng, min(new, most), most), new=min(new, most), ragged=rng.random() < 0.7,
                    window=rng.choice((0, 0, 0, 100, 4096)))
    batch = _log_int(rng, 1, 128)
    return dict(c, batch=batch, tokens=batch if rng.random() < 0.5 else max(batch, _log_int(rng, 16, 4096)), ctx=_log_int(rng, 1, 2000),
                turned=turned, interleaved=rng.randrange(2), factor=rng.choice((1.0, 4.0, 8.0)))


# ---------------------------------------------------------------------------
# what the case alone decides: lengths, chunks, and which pages a sequence has
# ---------------------------------------------------------------------------
def _spread(n):
    return [(0.5 + (i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]


def _lengths(n, ctx, ragged):
    """`n` lengths up to `ctx`; ragged: every length from 1 on about as often on a logarithmic and a linear scale."""
    if not ragged:
        return [ctx] * n
    some = [ctx ** x if i % 2 else 1 + (ctx - 1) * x for i, x in enumerate(_spread(n))]
    return [ctx] + [min(ctx, max(1, int(x))) for x in some[1:]]


def _pages(lens, page, spare):
    """(tables [n, width] with -1 behind a sequence's pages, refs) of sequences whose pages lie scattered over the pool."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = np.random.default_rng(total * 31 + page).permutation(total).astype(np.int32)
    tables = np.full((len(lens), max(need) + 1), -1, np.int32)
    refs, at = np.zeros(total, np.int32), 0
    for i, k in enumerate(need):
        tables[i, :k] = order[at:at + k]
        at += k
    refs[order[:at]] = 1
    return tables, refs


def _plan(case):
    """lens, tables, refs, and the lists that the call takes, as numpy arrays."""
    b = case["batch"]
    if case["kind"] == "chunk":
        lens = _lengths(b, case["ctx"], case["ragged"])
        new = [min(n, case["new"]) for n in lens]
        if case["ragged"] and case["new"] > 8:   # prompts of every length, every third sequence with one token
            new = [new[0]] + [1 if i % 3 == 2 else max(1, min(n, int(case["new"] ** u))) for i, (n, u) in enumerate(zip(lens, _spread(b)))][1:]
        tables, refs = _pages(lens, case["page"], 3)
        seqs, rows = list(range(b)), list(new)
        if b > 1:   # a captured step's padding
            seqs, rows = seqs + [-1], rows + [3]
        return dict(lens=lens, new=new, tables=tables, refs=refs, seqs=seqs, starts=np.cumsum([0] + rows))
    t = case["tokens"]
    starts = [x - 1 for x in _lengths(b, case["ctx"], True)]
    per = [t // b + (i < t % b) for i in range(b)]
    lens = [s + n for s, n in zip(starts, per)]
    tables, refs = _pages(lens, case["page"], 3)
    seqs = [i for i, n in enumerate(per) for _ in range(n)]
    return dict(lens=lens, tables=tables, refs=refs, seqs=seqs, pos=[s + j for s, n in zip(starts, per) for j in range(n)])


def _frequencies(case):
    """float64 [turned / 2]: radians per position; slow ones stretched by the factor, fast ones kept, a ramp between."""
    f = THETA ** (-np.arange(0, case["turned"], 2) / case["turned"])
    if case["factor"] == 1.0:
        return f
    turns = 8192 * f / (2 * math.pi)   # over the context that the model learned with
    keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
    return keep * f + (1 - keep) * f / case["factor"]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


def _gen(seed, stream):
    return torch.Generator("cuda").manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFF)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _pool(g, case, pages):
    shape = (pages, case["page"], case["kv"], case["hd"]) if case["order"] == "slot" else (pages, case["kv"], case["page"], case["hd"])
    dt, out = TYPES[case["dtype"]], torch.empty(2, *shape, device="cuda", dtype=TYPES[case["dtype"]])
    for i in range(2):
        out[i] = _randn(g, *shape, dtype=torch.float32 if case["dtype"] == "e4m3" else dt).to(dt)
    return out


def _cache(s, case, seed, p):
    g = _gen(seed, 1)
    s.k, s.v = (_pool(g, case, len(p["refs"])) for _ in range(2))
    s.scales = torch.exp(0.3 * _randn(g, 2, 2, case["kv"])) if case["dtype"] == "e4m3" else None
    s.refs, s.tables, s.lens, s.seqs = (_ints(p[x]) for x in ("refs", "tables", "lens", "seqs"))
    s.by_head, s.page, s.kv, s.hd, s.layer = case["order"] == "head", case["page"], case["kv"], case["hd"], 1
    s.heads, s.dtype, s.rows = case["heads"], case["dtype"], case["rows"]
    return g


def _rope_plan(s, case):
    s.turned, s.interleaved = case["turned"], case["interleaved"]
    s.freqs = torch.from_numpy(_frequencies(case)).cuda()
    s.factor = 1.0 if case["factor"] == 1.0 else float(np.float32(0.1 * math.log(case["factor"]) + 1.0))   # of cos and sin


def _prepare_logits(s, case, seed):
    g = _gen(seed, 2)
    n, v, h, b, m = (case[x] for x in ("batch", "vocab", "history", "bias", "masks"))
    s.rows, s.n_masks = case["rows"], m
    x = 2.5 * _randn(g, n, v + case["pad"])
    x[:, :v] += 6 * (_rand(g, n, v) < 8 / v)   # a few likely continuations
    s.logits = x.to(TYPES[s.rows])[:, :v]
    s.out = torch.empty_like(x, dtype=TYPES[s.rows])[:, :v]
    # text repeats itself: a history's tokens are a few hundred different ones, the common ones over and over
    words = _randint(g, 0, v, n, 400)
    s.history = torch.gather(words, 1, (400 * _rand(g, n, max(h, 1)) ** 3).long().clamp(max=399))
    s.lens = _ints([h if i % 4 == 0 else int(h * u) for i, u in enumerate(_spread(n))])
    s.prompt = s.lens // 3
    s.repetition, s.frequency, s.presence = 1 + 0.3 * _rand(g, n), 0.4 * _rand(g, n), 0.4 * _rand(g, n)
    s.repetition[::3] = 1.0
    per = [b if i % 2 == 0 else int(b * u) for i, u in enumerate(_spread(n))]
    s.starts = _ints(np.cumsum([0] + per))
    s.bias_ids, s.bias = _randint(g, 0, v, max(sum(per), 1)), 3 * _randn(g, max(sum(per), 1))
    s.bias_row = torch.from_numpy(np.repeat(np.arange(n), per)).cuda()   # (the plain form's)
    # a grammar's states: a handful of tokens, or most of them; every fourth row has none
    share = [0.5 if i % 2 else 0.002 for i in range(max(m, 1))]
    bits = torch.stack([_rand(g, v) < f for f in share]).cpu().numpy()
    words = np.zeros((max(m, 1), -(-v // 32) * 4), np.uint8)
    words[:, :-(-v // 8)] = np.packbits(bits, axis=1, bitorder="little")
    if m > 2:
        words[2] = 0   # a state that allows nothing
    s.masks = torch.from_numpy(words.view(np.int32)).cuda()
    s.mask_rows = _ints([-1 if m == 0 or i % 4 == 3 else i % m for i in range(n)])
    return s


def prepare(case, seed):
    s = _State()
    s.kind, s.handle = case["kind"], None
    if s.kind == "logits":
        return _prepare_logits(s, case, seed)
    if s.kind == "rope":
        g = _gen(seed, 3)
        s.rows, s.heads, s.hd = case["rows"], case["heads"], case["hd"]
        s.x = _randn(g, case["tokens"], s.heads, s.hd).to(TYPES[s.rows])
        s.out = torch.empty_like(s.x)
        s.pos = _ints([int(case["far"] * u) for u in _spread(case["tokens"])])
        _rope_plan(s, case)
        return s
    p = _plan(case)
    g = _cache(s, case, seed, p)
    n, h, kv, hd = int(p["starts"][-1]) if s.kind == "chunk" else len(p["seqs"]), s.heads, s.kv, s.hd
    if s.kind == "chunk":
        s.window, s.starts, s.most = case["window"], _ints(p["starts"]), int(max(np.diff(p["starts"])))
        s.q = (1.5 * _randn(g, n, h, hd)).to(TYPES[s.rows])
        s.out = torch.zeros_like(s.q)
        s.scale = 1.0 / math.sqrt(hd)
    else:
        s.pos = _ints(p["pos"])
        qkv = _randn(g, n, h + 2 * kv, hd).to(TYPES[s.rows])   # as one projection leaves them
        s.q, s.kn, s.vn = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        s.qr = torch.empty(n, h, hd, device="cuda", dtype=TYPES[s.rows])
        _rope_plan(s, case)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _pool_rows(s, pool, tables):
    """float32 [n, kv, positions, hd] of the sequences' pages."""
    x = pool[s.layer][tables]   # [n, width, page, kv, hd]
    if s.by_head:
        x = x.transpose(2, 3)
    return x.reshape(len(tables), -1, s.kv, s.hd).float().transpose(1, 2)


def _chunk(s):
    live = s.seqs >= 0
    seqs, starts = s.seqs.clamp(min=0).long(), s.starts.long()
    n, rows, g = len(seqs), len(s.q), s.heads // s.kv
    tables = s.tables[seqs].long().clamp(min=0)
    # row t of the call: token j of chunk i
    t = torch.arange(rows, device="cuda")
    i = torch.searchsorted(starts[1:], t, right=True)
    j = t - starts[i]
    q = torch.zeros(n, s.most, s.heads, s.hd, device="cuda")
    q[i, j] = s.q.float()
    q = q.view(n, s.most, s.kv, g, s.hd).permute(0, 2, 3, 1, 4).reshape(n, s.kv, g * s.most, s.hd)
    k, v = _pool_rows(s, s.k, tables), _pool_rows(s, s.v, tables)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    if s.scales is not None:
        x *= s.scales[0, s.layer][:, None, None]
    at = torch.arange(x.shape[-1], device="cuda")
    p = (s.lens[seqs] - (starts[1:] - starts[:-1]))[:, None, None] + torch.arange(s.most, device="cuda")[:, None]
    seen = at <= p   # [n, most, positions]
    if s.window:
        seen &= at > p - s.window
    x = x.view(n, s.kv, g, s.most, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    z = e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(e.view(n, s.kv, g * s.most, -1), v.contiguous()).view(n, s.kv, g, s.most, s.hd) / z
    if s.scales is not None:
        o *= s.scales[1, s.layer][:, None, None, None]
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s.most, s.heads, s.hd)[i, j]
    s.out.copy_(torch.where(live[i][:, None, None], o.to(s.out.dtype), s.out))
    return s.out


def _turned(s, x):
    """x [n, heads, hd] as float32, its first `turned` dims rotated by the positions' angles."""
    a = s.pos.double()[:, None, None] * s.freqs
    c, d = ((f(a) * s.factor).float() for f in (torch.cos, torch.sin))
    x = x.float()
    x, rest = x[..., :s.turned], x[..., s.turned:]
    if s.interleaved:
        u, w = x[..., 0::2], x[..., 1::2]
        y = torch.stack((u * c - w * d, u * d + w * c), -1).reshape(x.shape)
    else:
        u, w = x.chunk(2, -1)
        y = torch.cat((u * c - w * d, u * d + w * c), -1)
    return torch.cat((y, rest), -1)


def _rope(s):
    s.out.copy_(_turned(s, s.x))
    return s.out


def _append(s):
    seqs, pos = s.seqs.long(), s.pos.long()
    page, slot = s.tables[seqs, pos // s.page].long(), pos % s.page
    s.qr.copy_(_turned(s, s.q))
    for which, (pool, rows) in enumerate(((s.k, _turned(s, s.kn)), (s.v, s.vn.float()))):
        if s.scales is not None:
            rows = (rows / s.scales[which, s.layer][:, None]).clamp(-448.0, 448.0)
        to, rows = pool[s.layer].view(torch.uint8), rows.to(TYPES[s.dtype]).view(torch.uint8)   # (no scatter of 8-bit floats in torch)
        if s.by_head:
            to.transpose(1, 2)[page, slot] = rows
        else:
            to[page, slot] = rows
    return {"q": s.qr, "k": s.k, "v": s.v}


def _logits(s):
    n, v = s.logits.shape
    x = s.logits.float()
    at = torch.arange(s.history.shape[1], device="cuda")
    ids = s.history.long()
    one = (at < s.lens[:, None]).to(torch.int32)
    zeros = lambda: torch.zeros(n, v, device="cuda", dtype=torch.int32)  # noqa: E731
    seen = zeros().scatter_add_(1, ids, one) > 0
    count = zeros().scatter_add_(1, ids, one * (at >= s.prompt[:, None]))
    r = s.repetition[:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - s.frequency[:, None] * count - s.presence[:, None], x)
    last = int(s.bias_row.numel())   # a token listed twice has its last value
    place = torch.arange(1, last + 1, device="cuda", dtype=torch.int32)
    which = zeros().view(-1).scatter_reduce_(0, s.bias_row * v + s.bias_ids[:last].long(), place, "amax").view(n, v)
    x = torch.where(which > 0, x + s.bias[(which.long() - 1).clamp(min=0)], x)
    if s.n_masks:
        bits = (s.masks[..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.view(len(s.masks), -1)[:, :v] > 0
        none = (s.mask_rows < 0)[:, None]
        x = torch.where(none | allowed[s.mask_rows.clamp(min=0).long()], x, -math.inf)
    s.out.copy_(x)
    return s.out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _handle(s):
    """What a program keeps beside its buffers: descriptors, a workspace."""
    pkg = os.path.join(os.getcwd(), "gsd-lq_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from gsdlq import hip
    h = _State()
    h.lib, h.rows = hip.lib(), hip.ROW_TYPES[s.rows]
    if s.kind == "logits":
        h.rules = hip.GsdLogitRules(
            history=s.history.data_ptr(), history_lens=s.lens.data_ptr(), prompt_lens=s.prompt.data_ptr(), history_width=s.history.shape[1],
            repetition=s.repetition.data_ptr(), frequency=s.frequency.data_ptr(), presence=s.presence.data_ptr(),
            bias_starts=s.starts.data_ptr(), bias_ids=s.bias_ids.data_ptr(), bias=s.bias.data_ptr(), n_bias=len(s.bias))
        if s.n_masks:
            h.rules.masks, h.rules.mask_rows = s.masks.data_ptr(), s.mask_rows.data_ptr()
            h.rules.mask_words, h.rules.n_masks = s.masks.shape[1], len(s.masks)
        h.at = ctypes.byref(h.rules)
        return h
    if s.kind != "chunk":
        h.turn = hip.GsdRope(freqs=s.freqs.data_ptr(), rotary_dim=s.turned, interleaved=s.interleaved, scale=s.factor)
        h.rope = ctypes.byref(h.turn)
    if s.kind == "rope":
        return h
    scale = [None if s.scales is None else s.scales[i].data_ptr() for i in range(2)]
    h.status = torch.zeros(1, device="cuda", dtype=torch.int32)
    h.cache = hip.GsdPagedCache(
        k=s.k.data_ptr(), v=s.v.data_ptr(), k_scale=scale[0], v_scale=scale[1], refs=s.refs.data_ptr(),
        tables=s.tables.data_ptr(), lens=s.lens.data_ptr(), status=h.status.data_ptr(), n_layers=s.k.shape[0],
        n_pages=s.k.shape[1], page_size=s.page, n_kv_heads=s.kv, head_dim=s.hd, dtype=hip.KV_TYPES[s.dtype],
        head_major=int(s.by_head), n_seqs=s.tables.shape[0], table_width=s.tables.shape[1])
    h.at = ctypes.byref(h.cache)
    if s.kind == "chunk":
        need = h.lib.gsdh_paged_chunk_attention_workspace_bytes(h.at, len(s.seqs), len(s.q), s.heads)
        h.space = torch.zeros(max(int(need), 4), device="cuda", dtype=torch.uint8)
    return h


def _own(s):
    if s.handle is None:
        s.handle = _handle(s)
    h, lib, st = s.handle, s.handle.lib, torch.cuda.current_stream().cuda_stream
    if s.kind == "logits":
        lib.gsdh_logits_adjust(st, h.at, s.logits.data_ptr(), h.rows, s.logits.stride(0), *s.logits.shape, s.out.data_ptr(), s.out.stride(0))
        return s.out
    if s.kind == "rope":
        lib.gsdh_rope_rows(st, h.rope, s.x.data_ptr(), h.rows, s.x.stride(0), s.out.data_ptr(), s.out.stride(0), s.pos.data_ptr(), len(s.x),
                           s.heads, s.hd)
        return s.out
    if s.kind == "append":
        lib.gsdh_paged_rope_append(st, h.at, s.layer, h.rope, h.rows, s.q.data_ptr(), s.q.stride(0), s.kn.data_ptr(), s.kn.stride(0),
                                   s.vn.data_ptr(), s.vn.stride(0), s.qr.data_ptr(), s.qr.stride(0), s.seqs.data_ptr(), s.pos.data_ptr(),
                                   len(s.seqs), s.heads)
        return {"q": s.qr, "k": s.k, "v": s.v}
    lib.gsdh_paged_chunk_attention(st, h.at, s.layer, s.q.data_ptr(), h.rows, s.q.stride(0), s.seqs.data_ptr(), s.starts.data_ptr(), len(s.seqs),
                                   len(s.q), s.heads, s.scale, s.window, s.out.data_ptr(), s.out.stride(0), h.space.data_ptr(),
                                   h.space.numel())
    return s.out


_PLAIN = {"chunk": _chunk, "rope": _rope, "append": _append, "logits": _logits}


def run(s):
    return _own(s) if own else _PLAIN[s.kind](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, rs = case["kind"], SIZE[case["rows"]]
    if kind == "logits":
        n, v, m = case["batch"], case["vocab"], case["masks"]
        at = [-1 if m == 0 or i % 4 == 3 else i % m for i in range(n)]
        # what a mask forbids need not be read
        read = sum(v if a < 0 else 0 if m > 2 and a == 2 else v * (0.5 if a % 2 else 0.002) for a in at)
        lists = sum(h if i % 4 == 0 else int(h * u) for i, u in enumerate(_spread(n)) for h in (case["history"],))
        return dict(bytes=int(rs * (read + n * v) + 4 * lists + 8 * n * case["bias"] * 3 // 4 + m * v // 8 + 32 * n), flops=n * v)
    if kind == "rope":
        n, h, hd = case["tokens"], case["heads"], case["hd"]
        return dict(bytes=2 * n * h * hd * rs + 4 * n + 4 * case["turned"], flops=3 * n * h * case["turned"])
    p, es = _plan(case), SIZE[case["dtype"]]
    h, kv, hd, ps = case["heads"], case["kv"], case["hd"], case["page"]
    row = 2 * es * kv * hd   # K and V of one position and layer
    if kind == "append":
        n = len(p["seqs"])
        return dict(bytes=n * (rs * hd * (2 * h + 2 * kv) + row + 12) + 4 * case["turned"], flops=3 * n * case["turned"] * (h + kv))
    b = f = 0
    for n, m in zip(p["lens"], p["new"]):
        w = case["window"] or n
        lowest = max(0, n - m + 1 - w)
        b += row * (n - lowest) + 2 * rs * m * h * hd + 4 * -(-(n - lowest) // ps)
        f += 4 * h * hd * sum(min(x, w) for x in range(n - m + 1, n + 1))
    return dict(bytes=b, flops=f)


# ---------------------------------------------------------------------------
# the operators' definitions, in 64 bits
# ---------------------------------------------------------------------------
def _rows_of(s, pool, which, seq, positions):
    """float64 [positions, kv, hd] of one sequence, its scale applied."""
    pos = torch.as_tensor(positions, device="cuda", dtype=torch.long)
    page, slot = s.tables[seq].long()[pos // s.page], pos % s.page
    x = pool[s.layer][page, :, slot] if s.by_head else pool[s.layer][page, slot]
    return x.double() if s.scales is None else x.double() * s.scales[which, s.layer].double()[:, None]


def _exact_chunk(s):
    out, starts, g = s.out.double(), s.starts.tolist(), s.heads // s.kv
    for i, seq in enumerate(s.seqs.tolist()):
        t0, t1 = starts[i], starts[i + 1]
        if seq < 0 or t1 == t0:
            continue
        n = int(s.lens[seq])
        k, v = _rows_of(s, s.k, 0, seq, range(n)), _rows_of(s, s.v, 1, seq, range(n))
        p = torch.arange(n - (t1 - t0), n, device="cuda")[:, None]
        back = p - torch.arange(n, device="cuda")
        hidden = (back < 0) | (back >= (s.window or n))
        for h in range(s.heads):
            x = s.q[t0:t1, h].double() @ k[:, h // g].T / math.sqrt(s.hd)
            out[t0:t1, h] = x.masked_fill_(hidden, -math.inf).softmax(-1) @ v[:, h // g]
    return out


def _exact_turn(s, x):
    x = x.double()
    r = s.turned
    angle = torch.polar(torch.full((1,), s.factor, device="cuda", dtype=torch.float64), (s.pos.double()[:, None] * s.freqs))[:, None]
    z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) if s.interleaved else torch.complex(x[..., :r // 2], x[..., r // 2:r])
    z = z * angle
    y = x.clone()
    y[..., :r] = torch.view_as_real(z).flatten(-2) if s.interleaved else torch.cat((z.real, z.imag), -1)
    return y


def _exact_append(s):
    k, v = s.k.double(), s.v.double()
    pos, tables = s.pos.tolist(), s.tables.tolist()
    page = torch.tensor([tables[a][b // s.page] for a, b in zip(s.seqs.tolist(), pos)], device="cuda")
    slot = torch.tensor([b % s.page for b in pos], device="cuda")
    for which, (pool, rows) in enumerate(((k, _exact_turn(s, s.kn)), (v, s.vn.double()))):
        if s.scales is not None:
            rows = rows / s.scales[which, s.layer].double()[:, None]
        (pool[s.layer].transpose(1, 2) if s.by_head else pool[s.layer])[page, slot] = rows
    return {"q": _exact_turn(s, s.q), "k": k, "v": v}


def _exact_logits(s):
    out = s.logits.cpu().double().numpy().copy()
    history, lens, prompt, starts = s.history.cpu().numpy(), s.lens.tolist(), s.prompt.tolist(), s.starts.tolist()
    ids, bias = s.bias_ids.tolist(), s.bias.double().tolist()
    rep, freq, pres = (t.double().tolist() for t in (s.repetition, s.frequency, s.presence))
    masks, rows = s.masks.cpu().numpy().view(np.uint8), s.mask_rows.tolist()
    for i in range(len(out)):
        y = out[i]
        seen = np.unique(history[i, :lens[i]])
        y[seen] = np.where(y[seen] > 0, y[seen] / rep[i], y[seen] * rep[i])
        said, count = np.unique(history[i, prompt[i]:lens[i]], return_counts=True)
        y[said] -= freq[i] * count + pres[i]
        for t, b in dict(zip(ids[starts[i]:starts[i + 1]], bias[starts[i]:starts[i + 1]])).items():
            y[t] += b
        if rows[i] >= 0:
            y[np.unpackbits(masks[rows[i]], bitorder="little")[:len(y)] == 0] = -math.inf
    return torch.from_numpy(out)


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "chunk":
        return _exact_chunk(s)
    if s.kind == "rope":
        return _exact_turn(s, s.x)
    return _exact_append(s) if s.kind == "append" else _exact_logits(s)
