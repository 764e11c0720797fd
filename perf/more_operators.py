"""Operators of serving from an 8-bit paged cache and of checking trees of drafted tokens.

  store    the new rows of a batch, from raw [Q | K | V] projections: per-head norm and rotary positions,
           keys and values quantised to 8 bits (e4m3 or int8, one scale per head and row) into the
           sequences' pages; the normed queries
  load     cached rows read back as 32-bit values
  attend   the batch's new rows (single tokens, drafts, chunks of prompts) over the 8-bit pages
  tree     each sequence's new rows are a tree of drafted tokens: a row sees the cache before them and its
           ancestors; over the 32-bit pool or the 8-bit one
  keep     the cache rows of an accepted path move together behind the context, and the lengths follow

Each case is one pass of one layer.  The plan of a batch follows from its lengths alone and serves every
layer of a forward pass, so it is made in `prepare`.  Heads of 128 values, 32-bit queries and outputs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
EPS = 1e-6
THETA = 1e6
SCALE = 1.0 / math.sqrt(D)
MOST = {"int8": 127.0, "e4m3": 448.0}  # the largest code


def listed():
    return [
        # one token of each of 48 conversations
        dict(name="store_tokens", kind="store", cache="e4m3", heads=16, kv_heads=8, block=64,
             lens=" ".join(["1"] * 48), past=" ".join(str(17 + 131 * i) for i in range(48))),
        # two whole prompts and a chunk late in a third, of a 4B-shaped layer
        dict(name="store_prompts", kind="store", cache="int8", heads=32, kv_heads=8, block=128,
             lens="2048 1500 4096", past="0 0 6000"),
        # the last rows of a few conversations, handed to a program that wants them in 32 bits
        dict(name="load_tails", kind="load", cache="e4m3", heads=16, kv_heads=8, block=32,
             lens="37 300 1 129 64", past="100 0 4999 777 2000"),
        # whole sequences, for instance before they are sent to another machine
        dict(name="load_long", kind="load", cache="int8", heads=32, kv_heads=8, block=128,
             lens="32768 9001 20000", past="0 0 0"),
        # single tokens of a ragged serving batch
        dict(name="attend_tokens", kind="attend", cache="e4m3", heads=32, kv_heads=8, block=64,
             lens=" ".join(["1"] * 24),
             past="255 8000 412 3333 1024 6200 90 2047 5120 700 31 4096 "
                  "1500 7777 2600 63 880 4999 300 1900 6500 128 2222 50"),
        # one token far into a very long context, five query heads to a KV head
        dict(name="attend_long", kind="attend", cache="int8", heads=40, kv_heads=8, block=128, lens="1",
             past="130001"),
        # a chunk of a prompt late in it, with running conversations beside it
        dict(name="attend_chunk", kind="attend", cache="int8", heads=32, kv_heads=8, block=64, lens="1024 1 1 5",
             past="12000 3000 777 6001"),
        # small trees over the 32-bit pool
        dict(name="tree_small", kind="tree", cache="f32", heads=16, kv_heads=8, block=32, lens="13 7 13 9 13 1",
             past="1000 333 64 2047 500 90"),
        # the usual size of a tree, a serving batch over the 8-bit pool
        dict(name="tree_serving", kind="tree", cache="e4m3", heads=32, kv_heads=8, block=64,
             lens=" ".join(["48"] * 16), past=" ".join(str(1500 + 311 * i) for i in range(16))),
        # wide trees over long contexts in the 32-bit pool
        dict(name="tree_wide", kind="tree", cache="f32", heads=32, kv_heads=8, block=128, lens="64 61 100",
             past="16000 9000 4321"),
        # accepted paths of a few small trees
        dict(name="keep_small", kind="keep", cache="f32", heads=16, kv_heads=8, block=32, lens="13 7 13 9 13 1",
             past="1000 333 64 2047 500 90"),
        # accepted paths of a serving batch of wide trees
        dict(name="keep_serving", kind="keep", cache="int8", heads=32, kv_heads=8, block=64,
             lens=" ".join(["64"] * 48), past=" ".join(str(100 + 57 * i) for i in range(48))),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "load", "attend", "attend", "attend", "tree", "tree", "tree", "keep"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (40, 8), (64, 8), (8, 8), (8, 2)])
    cache = rng.choice(["e4m3", "int8"] if kind in ("store", "load", "attend") else ["f32", "e4m3", "int8"])
    if kind in ("store", "load"):
        n_seq = _log_int(rng, 1, 64)
        most = (7000 * 48 if kind == "store" else 60000 * 8) // (heads + 2 * kv_heads if kind == "store" else kv_heads)
        lens = [_log_int(rng, 1, max(1, most // n_seq)) for _ in range(n_seq)]
        past = [rng.choice([0, _log_int(rng, 1, 2000)]) for _ in lens]
    elif kind == "keep":
        lens = [_log_int(rng, 1, 128) for _ in range(_log_int(rng, 1, 64))]
        past = [_log_int(rng, 1, 3000) for _ in lens]
    else:
        style = rng.choice(["token", "tokens", "drafts"] if kind == "attend" else ["one", "few", "batch"])
        if rng.random() < 0.25 and kind == "attend":
            style = "chunk"
        n_seq = {"token": 1, "one": 1, "chunk": rng.randrange(1, 4), "few": rng.randrange(2, 6)}.get(
            style, _log_int(rng, 2, 32))
        lens = [{"token": 1, "tokens": 1, "drafts": rng.randrange(1, 9)}.get(
            style, _log_int(rng, 30, 1000) if style == "chunk" else _log_int(rng, 2, 128)) for _ in range(n_seq)]
        longest = {"token": 100000, "one": 30000, "chunk": 12000, "few": 16000}.get(style, 8000)
        past = [rng.choice([_log_int(rng, 1, 500), _log_int(rng, 30, longest)]) for _ in lens]
        # no more pairs than in the largest listed case, nor scores where the plain form pads every sequence to the largest
        while (sum(n * (p + n) for n, p in zip(lens, past)) * heads > 1024 * 12000 * 32 or sum(past) > 130000 or
               n_seq * max(lens) * (max(past) + max(lens)) * heads > 4 * 1024 * 13024 * 32):
            past = [p // 2 for p in past]
    return dict(kind=kind, cache=cache, heads=heads, kv_heads=kv_heads, block=rng.choice([32, 64, 128, 256]),
                lens=" ".join(map(str, lens)), past=" ".join(map(str, past)))


# ------------------------------------------------------------------------------ inputs
def _ints(text):
    return [int(x) for x in text.split()]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _quantise(x, cache):
    """Head rows [..., 128] -> codes, scales [...]: the operations of the format's definition in their order, since a
    code is a step function of them."""
    a = x.abs().amax(-1)
    top = torch.tensor(MOST[cache], dtype=torch.float64, device=x.device)
    s, inv = (a.double() / top).float(), (top / a.double()).float()  # (each rounded once: a 32-bit division)
    small, bad = a < 2.0 ** -110, ~torch.isfinite(a)
    inv = torch.where(small | bad, torch.zeros_like(inv), inv)
    s = torch.where(small, torch.zeros_like(s), torch.where(bad, torch.full_like(s, math.nan), s))
    y = torch.where(bad[..., None], torch.zeros_like(x), x) * inv[..., None]
    return y.round().to(torch.int8) if cache == "int8" else y.to(torch.float8_e4m3fn), s


def _tree(rng, n):
    """Ancestor bits (its own among them) of n drafted tokens, parents before children."""
    bits = []
    for i in range(n):
        parent = -1 if i == 0 else rng.randrange(max(-1, i - 12), i)
        bits.append((1 << i) | (bits[parent] if parent >= 0 else 0))
    return bits


def _words(bits, words):
    """Ancestor bits as signed 64-bit words."""
    out = []
    for w in range(words):
        x = (bits >> (64 * w)) & (2 ** 64 - 1)
        out.append(x - 2 ** 64 if x >= 2 ** 63 else x)
    return out


def _kept(rng, n):
    """The accepted path: its first tokens in place, the others further back than it is long, as in a tree that is
    laid out level by level (a pass repeated on what it moved then moves the same rows)."""
    m = rng.randrange(0, min(n, 9) + 1)
    first = rng.randrange(0, m + 1)
    if n - m < m - first:
        first = m
    return list(range(first)) + sorted(rng.sample(range(m, n), m - first))


def _batch(c, seed):
    g, rng = _gen(seed), random.Random(seed)
    H, HKV, bs = c["heads"], c["kv_heads"], c["block"]
    lens, past = _ints(c["lens"]), _ints(c["past"])
    total = [p + n for p, n in zip(past, lens)]
    rows, starts = sum(lens), [sum(lens[:i]) for i in range(len(lens) + 1)]
    s = dict(c=c, lens=lens, past=past, starts=starts, rows=rows, max_kv=max(total))
    s["cu"], s["kv_len"] = _int32(starts), _int32(total)
    need = [(t + bs - 1) // bs for t in total]
    order = torch.randperm(sum(need), generator=g, device="cuda").tolist()
    table, at = torch.zeros((len(lens), max(need)), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.cuda()
    s["pages"] = sum(need)
    # the sequence of each row, its number among its sequence's rows, and where the new rows stand
    s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))
    s["i"] = torch.arange(rows, device="cuda") - s["cu"].long()[s["seq"]]
    s["slot"] = torch.tensor(past, device="cuda")[s["seq"]] + s["i"]

    def values(*shape):  # rows of uneven magnitude
        return _normal(g, *shape) * torch.exp(0.4 * _normal(g, *shape[:-1], 1))

    if c["kind"] == "store":
        s["qkv"] = values(rows, H + 2 * HKV, D).flatten(1)
        s["q_gamma"], s["k_gamma"] = 1.0 + 0.1 * _normal(g, D), 1.0 + 0.1 * _normal(g, D)
        f = THETA ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") / (D // 2))
        th = torch.arange(max(total), device="cuda").double()[:, None] * f
        s["cs"] = torch.stack([torch.cos(th).float(), torch.sin(th).float()], -1).contiguous()
    else:
        s["q"] = _normal(g, rows, H, D)
    if c["cache"] == "f32":
        s["k"], s["v"] = values(s["pages"] * bs, HKV, D), values(s["pages"] * bs, HKV, D)
    else:
        s["k"], s["k_scale"] = _quantise(values(s["pages"], HKV, bs, D), c["cache"])
        s["v"], s["v_scale"] = _quantise(values(s["pages"], HKV, bs, D), c["cache"])
    if c["kind"] == "tree":
        words = (max(lens) + 63) // 64
        bits = [b for n in lens for b in _tree(rng, n)]
        s["mask"] = torch.tensor([_words(b, words) for b in bits], dtype=torch.int64, device="cuda")
    if c["kind"] == "keep":
        kept = [_kept(rng, n) for n in lens]
        most = max(max(len(k) for k in kept), 1)
        s["kept"] = _int32([k + [-1] * (most - len(k)) for k in kept])
        s["n_kept"] = _int32([len(k) for k in kept])
        s["new_len"] = torch.zeros_like(s["kv_len"])
    if c["kind"] == "load":
        s["out"] = tuple(torch.empty((rows, HKV, D), dtype=torch.float32, device="cuda") for _ in range(2))
    elif c["kind"] != "keep":
        s["out"] = torch.empty((rows, H, D), dtype=torch.float32, device="cuda")
    return s


def prepare(case, seed):
    s = _batch(case, seed)
    if own:  # what a program keeps: the heads' shape, the pool's description, the plan of the forward pass
        from exactinfer_amd import attention as A

        s["shape"] = A.AttnShape(case["heads"], case["kv_heads"])
        s["batch"] = A.PackedBatch(len(s["lens"]), s["rows"], case["heads"], case["kv_heads"])
        s["batch"].plan(s["cu"], s["rows"], s["max_kv"], kv_len=s["kv_len"])
        if case["cache"] != "f32":
            s["cache"] = A.Cache8.of(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------------------------ plain forms
def _place(s, seq, t):
    """Page and row in it of keys t of sequences seq."""
    bs = s["c"]["block"]
    return s["table"][seq, t // bs].long(), t % bs


def _rows_at(s, name, page, at):
    """Cached head rows [..., HKV, 128] in 32 bits."""
    if s["c"]["cache"] == "f32":
        return s[name][page * s["c"]["block"] + at]
    return s[name][page, :, at].float() * s[name + "_scale"][page, :, at][..., None]


def _norm_turn(x, gamma, co, si):
    ss = x.double().pow(2).sum(-1, keepdim=True)
    eps = torch.tensor(EPS, dtype=torch.float32, device=x.device).double()
    y = x * (1.0 / torch.sqrt(ss / D + eps)).float() * gamma
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * co - b * si, a * si + b * co], -1)


def _plain_store(s):
    c = s["c"]
    H, HKV = c["heads"], c["kv_heads"]
    x = s["qkv"].view(s["rows"], H + 2 * HKV, D)
    co, si = s["cs"][s["slot"], :, 0][:, None], s["cs"][s["slot"], :, 1][:, None]
    q = _norm_turn(x[:, :H], s["q_gamma"], co, si)
    k, k_scale = _quantise(_norm_turn(x[:, H:H + HKV], s["k_gamma"], co, si), c["cache"])
    v, v_scale = _quantise(x[:, H + HKV:], c["cache"])
    page, at = _place(s, s["seq"], s["slot"])
    page, at, head = page[:, None], at[:, None], torch.arange(HKV, device="cuda")
    s["k"].view(torch.int8)[page, head, at] = k.view(torch.int8)
    s["v"].view(torch.int8)[page, head, at] = v.view(torch.int8)
    s["k_scale"][page, head, at], s["v_scale"][page, head, at] = k_scale, v_scale
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attend(s):
    """Every sequence padded to the longest, its rows to the most."""
    c = s["c"]
    H, HKV, S = c["heads"], c["kv_heads"], len(s["lens"])
    G, n, T = H // HKV, max(s["lens"]), s["max_kv"]
    t = torch.arange(T, device="cuda")
    seq = torch.arange(S, device="cuda")[:, None]
    page, at = _place(s, seq, t.expand(S, T))
    k = _rows_at(s, "k", page, at).permute(0, 2, 3, 1).contiguous()  # [S, HKV, 128, T]
    v = _rows_at(s, "v", page, at).permute(0, 2, 1, 3).contiguous()
    i = torch.arange(n, device="cuda")
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    row = (s["cu"][:-1].long()[:, None] + torch.minimum(i, lens[:, None] - 1))  # [S, n]
    q = s["q"][row].view(S, n, HKV, G, D).permute(0, 2, 3, 1, 4).reshape(S, HKV, G * n, D)
    w = (torch.matmul(q, k) * SCALE).view(S, HKV, G, n, T)
    first = (s["kv_len"].long() - lens)[:, None, None]
    j = t - first  # [S, 1, T]: the key's number among the new ones
    seen = j <= i[:, None]
    if c["kind"] == "tree":
        word = s["mask"][row].gather(2, (j.clamp(min=0) // 64).clamp(max=s["mask"].shape[1] - 1).expand(S, n, T))
        seen = seen & ((j < 0) | ((word >> (j.clamp(min=0) % 64)) & 1).bool())
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w -= w.amax(-1, keepdim=True)
    w.exp_()
    o = torch.matmul(w.view(S, HKV, G * n, T), v) / w.sum(-1).view(S, HKV, G * n, 1)
    return o.view(S, HKV, G, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, H, D)[s["seq"], s["i"]]


def _plain_keep(s):
    j = torch.arange(s["kept"].shape[1], device="cuda")[None]
    first = (s["kv_len"] - (s["cu"][1:] - s["cu"][:-1]))[:, None].long()
    valid = j < s["n_kept"][:, None]
    seq = torch.arange(len(s["lens"]), device="cuda")[:, None].expand_as(s["kept"])
    # rows that are not kept are written to themselves
    src = torch.where(valid, first + s["kept"], first)
    dst = torch.where(valid, first + j, first)
    src = torch.where(valid | (s["n_kept"][:, None] == 0), src, first + s["kept"][:, :1])
    p0, a0 = _place(s, seq, src)
    p1, a1 = _place(s, seq, dst)
    if s["c"]["cache"] == "f32":
        bs = s["c"]["block"]
        s["k"][p1 * bs + a1] = s["k"][p0 * bs + a0]
        s["v"][p1 * bs + a1] = s["v"][p0 * bs + a0]
    else:
        k, v = s["k"].view(torch.int8), s["v"].view(torch.int8)
        k[p1, :, a1], v[p1, :, a1] = k[p0, :, a0], v[p0, :, a0]
        s["k_scale"][p1, :, a1] = s["k_scale"][p0, :, a0]
        s["v_scale"][p1, :, a1] = s["v_scale"][p0, :, a0]
    s["new_len"] = (first[:, 0] + s["n_kept"]).to(torch.int32)
    return _state_out(s)


def _state_out(s):
    out = {"k": s["k"], "v": s["v"], "len": s["new_len"]}
    return out if s["c"]["cache"] == "f32" else {**out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain(s):
    kind = s["c"]["kind"]
    if kind == "store":
        return _plain_store(s)
    if kind == "load":
        page, at = _place(s, s["seq"], s["slot"])
        return _rows_at(s, "k", page, at), _rows_at(s, "v", page, at)
    return _plain_keep(s) if kind == "keep" else _plain_attend(s)


# ------------------------------------------------------------------------------ the framework's calls
def _calls(s):
    from exactinfer_amd import attention as A

    c, b = s["c"], s["batch"]
    if c["kind"] == "store":
        q = A.cache8_store(s["qkv"], s["cache"], s["table"], b, s["shape"], s["q_gamma"], s["k_gamma"], s["cs"],
                           out=s["out"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["kind"] == "load":
        return A.cache8_load(s["cache"], s["table"], b, out=s["out"])
    if c["kind"] == "keep":
        if c["cache"] == "f32":
            A.cache_keep(s["k"], s["v"], s["table"], c["block"], b, s["shape"], s["kept"], s["n_kept"],
                         out=s["new_len"])
        else:
            A.cache8_keep(s["cache"], s["table"], b, s["kept"], s["n_kept"], out=s["new_len"])
        return _state_out(s)
    if c["cache"] == "f32":
        return A.attn_tree_paged(s["q"], s["k"], s["v"], s["table"], c["block"], b, s["shape"], s["mask"],
                                 out=s["out"])
    return A.attn_packed_cache8(s["q"], s["cache"], s["table"], b, s["shape"], mask=s.get("mask"), out=s["out"])


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    H, HKV = c["heads"], c["kv_heads"]
    lens, past = _ints(c["lens"]), _ints(c["past"])
    rows, key = sum(lens), 2 * HKV * (4 * D if c["cache"] == "f32" else D + 4)  # bytes of a cached row
    if c["kind"] == "store":
        return {"bytes": rows * ((2 * H + 2 * HKV) * D * 4 + D * 4 + key),
                "flops": rows * (H + HKV) * D * 7 + 4 * rows * HKV * D}
    if c["kind"] == "load":
        return {"bytes": rows * (key + 2 * HKV * D * 4), "flops": rows * 2 * HKV * D}
    if c["kind"] == "keep":
        return {"bytes": sum(min(n, 9) for n in lens) // 2 * 2 * key, "flops": 0}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
    if c["kind"] == "tree":  # a row sees few of the other drafts
        pairs = sum(n * p + 4 * n for n, p in zip(lens, past))
    return {"bytes": 2 * rows * H * D * 4 + (sum(past) + rows) * key, "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------------------ in 64 bits
def _pages64(s, i, name, n):
    """The first n cached head rows of sequence i in 64 bits [n, HKV, 128]."""
    t = torch.arange(n, device="cuda")
    bs = s["c"]["block"]
    blk = s["table"][i].long().repeat_interleave(bs)[:n]
    if s["c"]["cache"] == "f32":
        return s[name].unflatten(0, (-1, bs))[blk, t % bs].double()
    codes = s[name].transpose(1, 2)[blk, t % bs].double()
    return codes * s[name + "_scale"].transpose(1, 2)[blk, t % bs].double()[..., None]


def _exact_attention(s):
    c, outs = s["c"], []
    H, HKV = c["heads"], c["kv_heads"]
    G = H // HKV
    for i, (n, p) in enumerate(zip(s["lens"], s["past"])):
        a, k, v = s["starts"][i], _pages64(s, i, "k", n + p), _pages64(s, i, "v", n + p)
        seen = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        if c["kind"] == "tree":
            words = s["mask"][a:a + n].tolist()
            bits = [sum((w % 2 ** 64) << (64 * x) for x, w in enumerate(r)) for r in words]
            seen = torch.tensor([[y <= x and bits[x] >> y & 1 == 1 for y in range(n)] for x in range(n)], device="cuda")
        out = torch.empty((n, H, D), dtype=torch.float64, device="cuda")
        for h in range(H):
            for b in range(0, n, 256):
                e = min(n, b + 256)
                w = torch.matmul(s["q"][a + b:a + e, h].double(), k[:, h // G].t().contiguous()) * SCALE
                w[:, p:][~seen[b:e]] = -math.inf
                out[b:e, h] = torch.matmul(torch.softmax(w, -1), v[:, h // G].contiguous())
        outs.append(out)
    return torch.cat(outs)


def _exact_store(s):
    c = s["c"]
    H, HKV, bs = c["heads"], c["kv_heads"], c["block"]
    q, k, v = s["qkv"].double().unflatten(-1, (-1, D)).split([H, HKV, HKV], 1)
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(s["past"], s["lens"])]).cuda()
    f = THETA ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * f)[:, None]

    def turned(x, gamma):
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * gamma.double()
        z = torch.view_as_real(torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn)
        return torch.cat([z[..., 0], z[..., 1]], -1)

    new = {"k": turned(k, s["k_gamma"]), "v": v}
    out = {"q": turned(q, s["q_gamma"])}
    page = torch.cat([s["table"][i].long().repeat_interleave(bs)[p:p + n]
                      for i, (n, p) in enumerate(zip(s["lens"], s["past"]))])
    for name in ("k", "v"):
        a = new[name].abs().amax(-1)
        scale = s[name + "_scale"].double()
        scale[page, :, pos % bs] = a / MOST[c["cache"]]
        out[name + "_scale"] = scale
        out[name] = None  # a whole number next to a border is that of the 32-bit value
        if c["cache"] == "e4m3":
            y = new[name] * (MOST["e4m3"] / a)[..., None]
            e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))  # steps of 2^(e - 3), of 2^-9 at the least
            step = torch.exp2(e - 3)
            codes = s[name].double()
            codes[page, :, pos % bs] = torch.round(y / step) * step
            out[name] = codes
    return out


def exact(case, seed):
    s = _batch(case, seed)
    kind = case["kind"]
    if kind == "store":
        return _exact_store(s)
    if kind == "load":
        return tuple(torch.cat([_pages64(s, i, name, n + p)[p:] for i, (n, p) in enumerate(zip(s["lens"], s["past"]))])
                     for name in ("k", "v"))
    if kind == "keep":
        return None  # rows are moved, nothing is computed
    return _exact_attention(s)
