"""What the paged cache's operators are measured on: attention of one new token
per sequence, RoPE with the append of K/V rows, forking and compacting pages,
and the log probabilities of tokens, each through the calls that a program
makes (the C ABI of `gsdlq.hip`), beside their plain forms in torch.

Head shapes are those of the benchmark and the tests, contexts go up to 131072
positions, vocabularies to some 130,000 entries.  The lengths of a ragged batch
and the pages of its sequences come from the case alone, every value from the
seed.
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


def listed():
    b = dict(heads=32, kv=8, hd=128, dtype="f16", page=16, order="slot")
    return [
        # the least a step can cost: one short sequence of the small test model
        dict(b, name="attend_short", kind="attend", heads=4, kv=2, hd=64, batch=1, ctx=33, ragged=False, window=0),
        # one user deep in a conversation
        dict(b, name="attend_8192", kind="attend", batch=1, ctx=8192, ragged=False, window=0),
        # a served batch: sequences of every length, an idle row behind them
        dict(b, name="attend_batch", kind="attend", batch=64, ctx=8191, ragged=True, window=0),
        # the same in 8 bits, pages by head, a sliding window over the older positions
        dict(b, name="attend_window_e4m3", kind="attend", dtype="e4m3", order="head", page=32, batch=48, ctx=9001,
             ragged=True, window=4096),
        # one document of 131072 positions
        dict(b, name="attend_long", kind="attend", dtype="bf16", page=64, batch=1, ctx=131072, ragged=False, window=0),
        # the rows of a decode step's new tokens
        dict(b, name="store_step", kind="store", batch=64, tokens=64, ctx=3000, interleaved=1),
        # chunks of several prompts in one call, 8-bit cache, rotation of halves
        dict(b, name="store_prompts", kind="store", dtype="e4m3", order="head", page=32, batch=5, tokens=4099, ctx=700,
             interleaved=0),
        # four prompts, each continued in eight ways
        dict(b, name="fork_branches", kind="fork", layers=32, parents=4, branches=8, ctx=1003),
        # half of the sequences of a long-running server have ended, the rest moves together
        dict(b, name="compact_half", kind="compact", layers=32, batch=24, ctx=700),
        # a sampled token's log probability and five alternatives
        dict(name="logprobs_token", kind="logprobs", rows=1, vocab=32768, dtype="f32", pad=0, top=5),
        # a text scored: every position's token
        dict(name="logprobs_text", kind="logprobs", rows=512, vocab=32768, dtype="f32", pad=0, top=1),
        # a batch's answers with many alternatives, a large odd vocabulary in 16 bits
        dict(name="logprobs_batch", kind="logprobs", rows=61, vocab=130001, dtype="bf16", pad=7, top=20),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "store", "fork", "compact", "logprobs", "logprobs"))
    if kind == "logprobs":
        vocab = _log_int(rng, 257, 140000)
        rows = _log_int(rng, 1, min(2048, 16000000 // vocab))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(("f32", "f32", "bf16", "f16")),
                    pad=rng.choice((0, 0, 1, 8)), top=rng.choice((0, 1, 5, 20, 32)))
    heads, kv, hd = rng.choice(HEADS)
    c = dict(kind=kind, heads=heads, kv=kv, hd=hd, dtype=rng.choice(("f16", "f16", "bf16", "e4m3")),
             page=rng.choice((8, 16, 16, 32, 64, 128)), order=rng.choice(("slot", "slot", "head")))
    if kind == "attend":
        batch = _log_int(rng, 1, 128)
        most = min(131072, 131072 * 1024 // (kv * hd * batch))
        return dict(c, batch=batch, ctx=_log_int(rng, 1, most), ragged=rng.random() < 0.7,
                    window=rng.choice((0, 0, 0, 100, 4096)))
    if kind == "store":
        batch = _log_int(rng, 1, 128)
        return dict(c, batch=batch, tokens=batch if rng.random() < 0.5 else max(batch, _log_int(rng, 16, 4096)),
                    ctx=_log_int(rng, 1, 2000), interleaved=rng.randrange(2))
    layers = rng.choice((2, 8, 32))
    if kind == "fork":
        return dict(c, layers=layers, parents=rng.randrange(1, 7), branches=rng.randrange(1, 9), ctx=_log_int(rng, 1, 1000))
    return dict(c, layers=layers, batch=rng.randrange(2, 25), ctx=_log_int(rng, 16, 700))


# ---------------------------------------------------------------------------
# what the case alone decides: lengths, and which pages a sequence has
# ---------------------------------------------------------------------------
def _lengths(n, ctx, ragged):
    """`n` lengths up to `ctx`; ragged: every length from 1 on about as often on a logarithmic and a linear scale."""
    if not ragged:
        return [ctx] * n
    u = [(0.5 + (i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]
    some = [ctx ** x if i % 2 else 1 + (ctx - 1) * x for i, x in enumerate(u)]
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
    kind = case["kind"]
    if kind == "attend":
        lens = _lengths(case["batch"], case["ctx"], case["ragged"])
        tables, refs = _pages(lens, case["page"], 3)
        seqs = list(range(len(lens))) + [-1] * (case["batch"] > 1)
        return dict(lens=lens, tables=tables, refs=refs, seqs=seqs)
    if kind == "store":
        b, t = case["batch"], case["tokens"]
        starts = [x - 1 for x in _lengths(b, case["ctx"], True)]
        per = [t // b + (i < t % b) for i in range(b)]
        lens = [s + n for s, n in zip(starts, per)]
        tables, refs = _pages(lens, case["page"], 3)
        seqs = [i for i, n in enumerate(per) for _ in range(n)]
        return dict(lens=lens, tables=tables, refs=refs, seqs=seqs, pos=[s + j for s, n in zip(starts, per) for j in range(n)])
    if kind == "fork":
        p, b = case["parents"], case["branches"]
        lens = _lengths(p, case["ctx"], True)
        tables, refs = _pages(lens, case["page"], 2 * p * b + 3)
        tables = np.concatenate([tables, np.full((p * b, tables.shape[1]), -1, np.int32)])
        src = [i // b for i in range(p * b)]
        return dict(lens=lens + [0] * (p * b), tables=tables, refs=refs, src=src, dst=list(range(p, p + p * b)))
    lens = _lengths(case["batch"], case["ctx"], True)
    tables, refs = _pages(lens, case["page"], 3)
    return dict(lens=lens, tables=tables, refs=refs, done=list(range(0, len(lens), 2)))


def _moves(p):
    """(pages still in use, how many of them a compaction moves) once the sequences of `done` are gone."""
    refs = p["refs"].copy()
    for s in p["done"]:
        refs[p["tables"][s][p["tables"][s] >= 0]] -= 1
    used = int((refs > 0).sum())
    return used, int((refs[used:] > 0).sum())


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


def _gen(seed, stream):
    return torch.Generator("cuda").manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFF)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _pool(g, case, layers, pages):
    shape = (pages, case["page"], case["kv"], case["hd"]) if case["order"] == "slot" else (pages, case["kv"], case["page"], case["hd"])
    dt, out = TYPES[case["dtype"]], torch.empty(layers, *shape, device="cuda", dtype=TYPES[case["dtype"]])
    for i in range(layers):
        out[i] = _randn(g, *shape, dtype=torch.float32 if case["dtype"] == "e4m3" else dt).to(dt)
    return out


def _cache(s, case, seed, p, layers):
    """The pools and the state of the pages: refs, tables and lens in one buffer, as it is kept for a restart."""
    g = _gen(seed, 1)
    s.k, s.v = (_pool(g, case, layers, len(p["refs"])) for _ in range(2))
    s.scales = None
    if case["dtype"] == "e4m3":
        s.scales = torch.exp(0.3 * _randn(g, 2, layers, case["kv"]))
    s.state0 = _ints(np.concatenate([p["refs"], p["tables"].reshape(-1), p["lens"]]))
    s.state = s.state0.clone()
    n, (rows, width) = len(p["refs"]), p["tables"].shape
    s.refs, s.tables, s.lens = s.state[:n], s.state[n:n + rows * width].view(rows, width), s.state[n + rows * width:]
    s.by_head, s.page, s.kv, s.hd = case["order"] == "head", case["page"], case["kv"], case["hd"]
    s.heads, s.dtype = case["heads"], case["dtype"]
    return g


def prepare(case, seed):
    s = _State()
    s.kind, s.handle = case["kind"], None
    if s.kind == "logprobs":
        g = _gen(seed, 2)
        n, v = case["rows"], case["vocab"]
        x = 2.5 * _randn(g, n, v + case["pad"])
        x[:, :v] += 6 * (torch.rand(n, v, generator=g, device="cuda") < 8 / v)   # a few likely continuations
        x[torch.rand(n, v + case["pad"], generator=g, device="cuda") < 0.02] = -math.inf   # what a grammar rules out
        s.tokens = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        x[torch.arange(n, device="cuda"), s.tokens.long()] = 2.5 * _randn(g, n)
        s.logits, s.top, s.dtype = x.to(TYPES[case["dtype"]])[:, :v], case["top"], case["dtype"]
        return s
    p = _plan(case)
    g = _cache(s, case, seed, p, case.get("layers", 2))
    if s.kind == "attend":
        s.seqs, s.window, s.layer = _ints(p["seqs"]), case["window"], 1
        s.q = 1.5 * _randn(g, len(p["seqs"]), s.heads, s.hd)
        s.out = torch.zeros_like(s.q)
        s.scale = 1.0 / math.sqrt(s.hd)
    elif s.kind == "store":
        n, h, kv, hd = len(p["seqs"]), s.heads, s.kv, s.hd
        s.seqs, s.pos, s.layer, s.interleaved = _ints(p["seqs"]), _ints(p["pos"]), 1, case["interleaved"]
        qkv = _randn(g, n, h + 2 * kv, hd)   # as one projection leaves them
        s.q, s.kn, s.vn = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        s.qr = torch.empty(n, h, hd, device="cuda")
        s.angles = _angles(max(p["pos"]) + 1, hd)
    elif s.kind == "fork":
        s.src, s.dst = _ints(p["src"]), _ints(p["dst"])
        s.more = torch.ones_like(s.dst)
    else:
        s.done = _ints(p["done"])
    return s


def _angles(n, hd):
    """float32 [n, hd / 2, 2]: (cos, sin) of the angles that the engine's format rounds to float32."""
    freq = (1.0 / np.float32(THETA) ** (np.arange(0, hd, 2, dtype=np.float32) / np.float32(hd))).astype(np.float32)
    a = (np.arange(n, dtype=np.float32)[:, None] * freq).astype(np.float64)
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _scale(s, which):
    """[kv] of this layer, or one."""
    return 1.0 if s.scales is None else s.scales[which, s.layer]


def _attend(s):
    live = s.seqs >= 0
    rows = s.seqs.clamp(min=0).long()
    tables, lens = s.tables[rows].long().clamp(min=0), torch.where(live, s.lens[rows], 0)
    n, width = tables.shape
    at = torch.arange(width * s.page, device="cuda")
    seen = (at < lens[:, None]) & ((at >= lens[:, None] - s.window) if s.window else True)
    k, v = s.k[s.layer][tables], s.v[s.layer][tables]   # [n, width, page, kv, hd]
    if s.by_head:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    k = k.reshape(n, -1, s.kv, s.hd).float().permute(0, 2, 3, 1)
    v = v.reshape(n, -1, s.kv, s.hd).float().permute(0, 2, 1, 3)
    x = torch.matmul(s.q.view(n, s.kv, -1, s.hd), k) * s.scale
    if s.scales is not None:
        x = x * _scale(s, 0)[:, None, None]
    seen = seen[:, None, None]
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    v = torch.where(seen[:, :, 0, :, None], v, 0.0)
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    if s.scales is not None:
        o = o * _scale(s, 1)[:, None, None]
    s.out.copy_(torch.where(live[:, None, None], o.reshape(n, -1, s.hd), s.out))
    return s.out


def _rotated(s, x, a):
    """RoPE of x [n, heads, hd] with the angles a [n, hd / 2, 2]."""
    c, d = a[:, None, :, 0], a[:, None, :, 1]
    if s.interleaved:
        u, w = x[..., 0::2], x[..., 1::2]
        return torch.stack((u * c - w * d, u * d + w * c), -1).reshape(x.shape)
    u, w = x.chunk(2, -1)
    return torch.cat((u * c - w * d, u * d + w * c), -1)


def _rounded(s, x, which):
    if s.scales is not None:
        x = (x / _scale(s, which)[:, None]).clamp(-448.0, 448.0)
    return x.to(TYPES[s.dtype])


def _store(s):
    seqs, pos = s.seqs.long(), s.pos.long()
    page, slot = s.tables[seqs, pos // s.page].long(), pos % s.page
    a = s.angles[pos]
    s.qr.copy_(_rotated(s, s.q, a))
    for pool, rows in ((s.k, _rounded(s, _rotated(s, s.kn, a), 0)), (s.v, _rounded(s, s.vn, 1))):
        to, rows = pool[s.layer].view(torch.uint8), rows.view(torch.uint8)   # (no scatter of 8-bit floats in torch)
        if s.by_head:
            to.transpose(1, 2)[page, slot] = rows
        else:
            to[page, slot] = rows
    return {"q": s.qr, "k": s.k, "v": s.v}


def _free_pages(s):
    """The free pages in rising order, those in use behind them."""
    return torch.argsort((s.refs != 0).to(torch.int8), stable=True).to(torch.int32)


def _fork(s):
    s.state.copy_(s.state0)
    src, dst = s.src.long(), s.dst.long()
    n = s.lens[src]
    full, part = n // s.page, n % s.page
    col = torch.arange(s.tables.shape[1], device="cuda", dtype=torch.int32)
    new = _free_pages(s)[((part > 0).cumsum(0) - 1).clamp(min=0)]
    old = s.tables[src]
    last = (col == full[:, None]) & (part > 0)[:, None]
    shared = col < full[:, None]
    s.tables[dst] = torch.where(shared, old, torch.where(last, new[:, None], -1))
    s.lens[dst] = n
    s.refs.index_add_(0, old.clamp(min=0).reshape(-1), shared.to(torch.int32).reshape(-1))
    s.refs.index_add_(0, new, (part > 0).to(torch.int32))
    from_, to = old.gather(1, full[:, None].long())[:, 0].clamp(min=0)[part > 0].long(), new[part > 0].long()
    keep = torch.arange(s.page, device="cuda") < part[part > 0][:, None]
    keep = keep[:, None, :, None] if s.by_head else keep[:, :, None, None]
    for pool in (s.k, s.v):
        bits = pool.view(torch.uint8)
        bits[:, to] = torch.where(keep, bits[:, from_], bits[:, to])
    # a page for the next token where the last one is full
    n, more = s.lens[dst], s.more
    have = (n + s.page - 1) // s.page
    need = (n + more + s.page - 1) // s.page - have
    free = _free_pages(s)
    k = col - have[:, None]
    taken = (k >= 0) & (k < need[:, None])
    new = free[((need.cumsum(0) - need)[:, None] + k).clamp(0, len(free) - 1)]
    s.tables[dst] = torch.where(taken, new, s.tables[dst])
    s.refs.index_add_(0, new.reshape(-1), taken.to(torch.int32).reshape(-1))
    s.lens[dst] = n + more
    return {"refs": s.refs, "tables": s.tables, "lens": s.lens, "k": s.k, "v": s.v}


def _compact(s):
    s.state.copy_(s.state0)
    done = s.done.long()
    gone = s.tables[done]
    s.refs.index_add_(0, gone.clamp(min=0).reshape(-1), -(gone >= 0).to(torch.int32).reshape(-1))
    s.tables[done] = -1
    s.lens[done] = 0
    used = s.refs > 0
    n = used.sum()
    at = torch.arange(len(used), device="cuda")
    src, dst = (used & (at >= n)).nonzero()[:, 0], (~used & (at < n)).nonzero()[:, 0]
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    for pool in (s.k, s.v):
        bits = pool.view(torch.uint8)
        bits[:, dst] = bits[:, src]
    s.refs[dst] = s.refs[src]
    s.refs[src] = 0
    s.tables.copy_(torch.where(s.tables >= 0, to[s.tables.clamp(min=0)], s.tables))
    return {"refs": s.refs, "tables": s.tables, "lens": s.lens, "used": n.to(torch.int32).view(1), "k": s.k, "v": s.v}


def _logprobs(s):
    x = s.logits.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1)
    log_z = torch.log(z)
    at = s.tokens.long()[:, None]
    entropy = log_z - (e * torch.where(e > 0, d, 0.0)).sum(-1) / z
    value, ids = torch.sort(x, dim=-1, descending=True, stable=True)   # (ties: the lowest index)
    return {"logprob": d.gather(1, at)[:, 0] - log_z, "entropy": entropy, "ids": ids[:, :s.top].to(torch.int32).contiguous(),
            "top": (value[:, :s.top] - m - log_z[:, None]).contiguous()}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _handle(s):
    """What a program keeps beside its buffers: the descriptor of the cache, a workspace, the outputs."""
    pkg = os.path.join(os.getcwd(), "gsd-lq_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from gsdlq import hip
    h = _State()
    h.lib = hip.lib()
    zeros = lambda n: torch.zeros(max(int(n), 4), device="cuda", dtype=torch.uint8)  # noqa: E731
    if s.kind == "logprobs":
        n, v = s.logits.shape
        h.space = zeros(h.lib.gsdh_token_logprobs_workspace_bytes(n, v, s.top))
        f = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        h.out = {"logprob": f(n), "entropy": f(n), "ids": f(n, s.top).to(torch.int32), "top": f(n, s.top)}
        return h
    scale = [None if s.scales is None else s.scales[i].data_ptr() for i in range(2)]
    h.status = torch.zeros(1, device="cuda", dtype=torch.int32)
    h.cache = hip.GsdPagedCache(
        k=s.k.data_ptr(), v=s.v.data_ptr(), k_scale=scale[0], v_scale=scale[1], refs=s.refs.data_ptr(),
        tables=s.tables.data_ptr(), lens=s.lens.data_ptr(), status=h.status.data_ptr(), n_layers=s.k.shape[0],
        n_pages=s.k.shape[1], page_size=s.page, n_kv_heads=s.kv, head_dim=s.hd, dtype=hip.KV_TYPES[s.dtype],
        head_major=int(s.by_head), n_seqs=s.tables.shape[0], table_width=s.tables.shape[1])
    h.at = ctypes.byref(h.cache)
    if s.kind == "attend":
        h.space = zeros(h.lib.gsdh_paged_attention_workspace_bytes(h.at, len(s.seqs), s.heads))
    elif s.kind in ("fork", "compact"):
        h.space = zeros(h.lib.gsdh_pages_workspace_bytes(h.at))
        h.used = torch.zeros(1, device="cuda", dtype=torch.int32)
    return h


def _own(s):
    if s.handle is None:
        s.handle = _handle(s)
    h, lib, st = s.handle, s.handle.lib, torch.cuda.current_stream().cuda_stream
    if s.kind == "logprobs":
        o = h.out
        lib.gsdh_token_logprobs(st, s.logits.data_ptr(), {"f32": 0, "f16": 1, "bf16": 2}[s.dtype], s.logits.stride(0), *s.logits.shape,
                                s.tokens.data_ptr(), s.top, o["logprob"].data_ptr(), o["entropy"].data_ptr(),
                                o["ids"].data_ptr(), o["top"].data_ptr(), h.space.data_ptr(), h.space.numel())
        return o
    if s.kind == "attend":
        lib.gsdh_paged_attention(st, h.at, s.layer, s.q.data_ptr(), s.q.stride(0), s.seqs.data_ptr(), len(s.seqs), s.heads,
                                 s.scale, s.window, s.out.data_ptr(), s.out.stride(0), h.space.data_ptr(), h.space.numel())
        return s.out
    if s.kind == "store":
        lib.gsdh_paged_rope_store(st, h.at, s.layer, s.q.data_ptr(), s.q.stride(0), s.kn.data_ptr(), s.kn.stride(0),
                                  s.vn.data_ptr(), s.vn.stride(0), s.qr.data_ptr(), s.qr.stride(0), s.seqs.data_ptr(),
                                  s.pos.data_ptr(), len(s.seqs), s.heads, s.angles.data_ptr(), len(s.angles), s.interleaved)
        return {"q": s.qr, "k": s.k, "v": s.v}
    s.state.copy_(s.state0)
    if s.kind == "fork":
        lib.gsdh_pages_fork(st, h.at, s.src.data_ptr(), s.dst.data_ptr(), len(s.src), h.space.data_ptr(), h.space.numel())
        lib.gsdh_pages_take(st, h.at, s.dst.data_ptr(), s.more.data_ptr(), len(s.dst))
        return {"refs": s.refs, "tables": s.tables, "lens": s.lens, "k": s.k, "v": s.v}
    lib.gsdh_pages_free(st, h.at, s.done.data_ptr(), len(s.done))
    lib.gsdh_pages_compact(st, h.at, h.used.data_ptr(), h.space.data_ptr(), h.space.numel())
    return {"refs": s.refs, "tables": s.tables, "lens": s.lens, "used": h.used, "k": s.k, "v": s.v}


_PLAIN = {"attend": _attend, "store": _store, "fork": _fork, "compact": _compact, "logprobs": _logprobs}


def run(s):
    return _own(s) if own else _PLAIN[s.kind](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n, v, t = case["rows"], case["vocab"], case["top"]
        return dict(bytes=n * v * SIZE[case["dtype"]] + n * (4 + 8 + 8 * t), flops=4 * n * v)
    p, es = _plan(case), SIZE[case["dtype"]]
    h, kv, hd, ps = case["heads"], case["kv"], case["hd"], case["page"]
    row = 2 * es * kv * hd   # K and V of one position and layer
    if kind == "attend":
        seen = [min(n, case["window"] or n) for n in p["lens"]]
        return dict(bytes=sum(row * n + 8 * h * hd + 4 * -(-n // ps) for n in seen), flops=sum(4 * h * hd * n for n in seen))
    if kind == "store":
        n = len(p["seqs"])
        return dict(bytes=n * (4 * hd * (2 * h + 2 * kv) + row + 4 * hd + 12), flops=6 * n * hd * (h + kv) // 2)
    state = 4 * (len(p["refs"]) + sum(-(-n // ps) for n in p["lens"]) + len(p["lens"]))
    if kind == "fork":
        rows = [p["lens"][i] % ps for i in p["src"]]
        return dict(bytes=2 * case["layers"] * row * sum(rows) + state + 8 * sum(-(-p["lens"][i] // ps) for i in p["src"]), flops=0)
    return dict(bytes=2 * case["layers"] * row * ps * _moves(p)[1] + 2 * state, flops=0)


# ---------------------------------------------------------------------------
# the operators' definitions, in 64 bits
# ---------------------------------------------------------------------------
def _rows_of(s, pool, which, seq, positions):
    """float64 [positions, kv, hd] of one sequence, its scale applied."""
    pos = torch.as_tensor(positions, device="cuda", dtype=torch.long)
    page, slot = s.tables[seq].long()[pos // s.page], pos % s.page
    x = pool[s.layer][page, :, slot] if s.by_head else pool[s.layer][page, slot]
    return x.double() if s.scales is None else x.double() * s.scales[which, s.layer].double()[:, None]


def _exact_attend(s):
    out = s.out.double()
    for i, seq in enumerate(s.seqs.tolist()):
        n = int(s.lens[seq]) if seq >= 0 else 0
        if n == 0:
            continue
        seen = range(max(0, n - s.window) if s.window else 0, n)
        k, v = _rows_of(s, s.k, 0, seq, seen), _rows_of(s, s.v, 1, seq, seen)
        g = s.heads // s.kv
        for j in range(s.kv):
            x = s.q[i, j * g:(j + 1) * g].double() @ k[:, j].T / math.sqrt(s.hd)
            out[i, j * g:(j + 1) * g] = x.softmax(-1) @ v[:, j]
    return out


def _exact_store(s):
    pos = s.pos.tolist()
    angle = torch.view_as_complex(s.angles.double())[pos][:, None]

    def turned(x):
        x = x.double()
        half = x.shape[-1] // 2
        z = torch.complex(x[..., 0::2], x[..., 1::2]) if s.interleaved else torch.complex(x[..., :half], x[..., half:])
        z = z * angle
        return torch.view_as_real(z).reshape(x.shape) if s.interleaved else torch.cat((z.real, z.imag), -1)

    k, v = s.k.double(), s.v.double()
    for which, (pool, rows) in enumerate(((k, turned(s.kn)), (v, s.vn.double()))):
        if s.scales is not None:
            rows = rows / s.scales[which, s.layer].double()[:, None]
        tables = s.tables.tolist()
        page = torch.tensor([tables[a][b // s.page] for a, b in zip(s.seqs.tolist(), pos)], device="cuda")
        slot = torch.tensor([b % s.page for b in pos], device="cuda")
        (pool[s.layer].transpose(1, 2) if s.by_head else pool[s.layer])[page, slot] = rows
    return {"q": turned(s.q), "k": k, "v": v}


def _exact_pages(s, case):
    """The moved rows one after another, on page lists of the host; whole numbers have no such value."""
    p = _plan(case)
    refs, tables, lens = p["refs"].tolist(), p["tables"].tolist(), list(p["lens"])
    k, v = s.k.double(), s.v.double()
    moves = []
    if case["kind"] == "fork":
        for a, b in zip(p["src"], p["dst"]):
            rest = lens[a] % s.page
            if rest:
                new = refs.index(0)
                refs[new] = 1
                moves.append((tables[a][lens[a] // s.page], new, rest))
    else:
        for a in p["done"]:
            for x in tables[a][:-(-lens[a] // s.page)]:
                refs[x] -= 1
        used = sum(r > 0 for r in refs)
        holes = [i for i in range(used) if refs[i] == 0]
        moves = [(a, b, s.page) for a, b in zip([i for i in range(used, len(refs)) if refs[i] > 0], holes)]
    for pool in (k, v):
        for a, b, n in moves:
            if s.by_head:
                pool[:, b, :, :n] = pool[:, a, :, :n]
            else:
                pool[:, b, :n] = pool[:, a, :n]
    out = {"refs": None, "tables": None, "lens": None, "k": k, "v": v}
    return out if case["kind"] == "fork" else dict(out, used=None)


def _exact_logprobs(s):
    n = len(s.logits)
    out = {"logprob": torch.empty(n, dtype=torch.float64), "entropy": torch.empty(n, dtype=torch.float64), "ids": None,
           "top": torch.empty(n, s.top, dtype=torch.float64)}
    for i in range(n):
        x = s.logits[i].double()
        x = x - torch.logsumexp(x, 0)
        x, t = x.cpu(), int(s.tokens[i])
        out["logprob"][i] = x[t]
        y = x[x > -math.inf]
        out["entropy"][i] = -(y.exp() * y).sum()
        out["top"][i] = torch.sort(x, descending=True).values[:s.top]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "logprobs":
        return _exact_logprobs(s)
    if s.kind == "attend":
        return _exact_attend(s)
    if s.kind == "store":
        return _exact_store(s)
    return _exact_pages(s, case)
