"""Operators of a serving step over the new rows of several sequences.

  rope     rotary positions of packed rows: half and interleaved layouts, part of the head or all of
           it, with or without the per-head RMS norm, from a table scaled for long contexts
  packed   causal attention over whole prompts of different lengths, packed one after another
  chunks   each sequence's new rows (a chunk, or a single token) attend over its pages of a shared
           pool of K/V blocks
  step     the same from raw projections: QK-norm + rotary positions + append to the pool + attention

Each case is one pass of one layer.  Where a plan of the batch is made from its lengths (once for all
layers of a forward pass), making it is part of the pass.  Heads of 128 values, 32-bit values.
"""
from __future__ import annotations

import math

import torch

own = False

D = 128
EPS = 1e-6
SCALE = 1.0 / math.sqrt(D)
BUDGET = 1 << 28  # scores held at a time by the plain forms


def listed():
    return [
        # one token of each of 48 conversations, far apart in a long context
        dict(name="rope_tokens", kind="rope", rows=48, heads=32, kv_heads=8, rope_dim=128, layout="half",
             scaling="yarn", n_pos=65536, norm=True),
        # a part of each head, interleaved pairs, an odd number of rows, no norm
        dict(name="rope_interleaved_part", kind="rope", rows=1533, heads=40, kv_heads=8, rope_dim=64,
             layout="interleaved", scaling="ntk", n_pos=16384, norm=False),
        # every prompt row of a large batch of a 4B-shaped layer
        dict(name="rope_prompts", kind="rope", rows=16384, heads=32, kv_heads=8, rope_dim=128, layout="half",
             scaling="none", n_pos=16384, norm=True),
        # a few short messages
        dict(name="packed_short", kind="packed", heads=16, kv_heads=8, lens="37 1 96 5 64"),
        # prompts of very different lengths, five query heads to a KV head
        dict(name="packed_ragged", kind="packed", heads=40, kv_heads=8, lens="700 33 1501 128 2 940 311 64 1 450 77"),
        # the largest: a long document among ordinary prompts of a 4B-shaped layer
        dict(name="packed_long", kind="packed", heads=32, kv_heads=8, lens="8192 2048 300 1024 17 4096"),
        # single tokens of a ragged serving batch over a pool of shuffled pages
        dict(name="chunks_tokens", kind="chunks", heads=16, kv_heads=8, block=64,
             lens=" ".join(["1"] * 24),
             past="255 8000 412 3333 1024 6200 90 2047 5120 700 31 4096 "
                  "1500 7777 2600 63 880 4999 300 1900 6500 128 2222 50"),
        # short runs of draft tokens to be checked, behind a common prefix of 1024 tokens
        dict(name="chunks_drafts", kind="chunks", heads=32, kv_heads=8, block=32, shared=1024,
             lens=" ".join(["5"] * 16), past=" ".join(str(1024 + 37 * i) for i in range(16))),
        # a step that mixes running conversations with chunks of two new prompts
        dict(name="step_mixed", kind="step", heads=16, kv_heads=8, block=64,
             lens="1 1 512 1 1 1 300 1 1 1 1 1 1 1",
             past="2000 150 1536 6000 33 900 0 4100 777 64 2500 1234 17 3001"),
        # a chunk late in a very long prompt, with a fresh prompt beside it
        dict(name="step_long_chunk", kind="step", heads=32, kv_heads=8, block=128, lens="1024 400", past="30000 0"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "packed", "packed", "chunks", "chunks", "step", "step"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (32, 8), (40, 8), (64, 8), (8, 8), (8, 2)])
    if kind == "rope":
        heads, kv_heads = rng.choice([(8, 8), (32, 8), (40, 8), (64, 8), (8, 2)])
        return dict(kind=kind, rows=_log_int(rng, 1, 16384 * 40 // (heads + kv_heads) // 2), heads=heads,
                    kv_heads=kv_heads, rope_dim=rng.choice([128, 128, 32, 64, 96]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    n_pos=_log_int(rng, 512, 131072), norm=rng.random() < 0.5)
    most = 6e11 / (4 * D * heads)  # query-key pairs per head: less than the largest listed case
    lens, past = [], []
    style = rng.choice(["tokens", "short", "mixed", "long"])
    n_seq = {"tokens": _log_int(rng, 1, 64), "short": _log_int(rng, 1, 48), "mixed": _log_int(rng, 2, 32),
             "long": rng.randrange(1, 4)}[style]
    for i in range(n_seq):
        if kind == "packed":
            n = _log_int(rng, 1, {"tokens": 64, "short": 300, "mixed": 3000, "long": 8192}[style])
            p = 0
        else:
            n = {"tokens": 1, "short": rng.randrange(1, 17),
                 "mixed": 1 if rng.random() < 0.7 else _log_int(rng, 2, 700), "long": _log_int(rng, 100, 2048)}[style]
            p = rng.choice([0, _log_int(rng, 1, 500), _log_int(rng, 30, 8000), _log_int(rng, 1000, 30000)])
            if style != "long":
                p = min(p, 12000)
        if n * p + n * (n + 1) // 2 > most or sum(lens) + n > 16384 or sum(past) + p > 150000:
            n, p = 1 + n % 50, p % 1000
        most -= n * p + n * (n + 1) // 2
        lens.append(n)
        past.append(p)
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, lens=" ".join(map(str, lens)))
    if kind != "packed":
        c.update(block=rng.choice([32, 64, 128, 256]), past=" ".join(map(str, past)))
    return c


# ------------------------------------------------------------------------------ inputs
THETA = 1e6
TRAINED = 32768  # the context the frequencies were trained for
FACTOR = 4.0


def _ints(text):
    return [int(x) for x in text.split()]


def _frequencies(rope_dim, scaling):
    """rope_dim/2 frequencies in 64 bits, and the factor on cos and sin."""
    i = torch.arange(rope_dim // 2, dtype=torch.float64, device="cuda")
    theta, m = THETA, 1.0
    if scaling == "ntk":
        theta = THETA * FACTOR ** (rope_dim / (rope_dim - 2))
    f = theta ** (-2.0 * i / rope_dim)
    if scaling == "linear":
        f = f / FACTOR
    if scaling == "yarn":
        def pair(turns):  # the pair that makes this many turns over the trained context
            return rope_dim * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rope_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f / FACTOR * ramp + f * (1.0 - ramp)
        m = 0.1 * math.log(FACTOR) + 1.0
    return f, m


def _cos_sin(pos, rope_dim, scaling):
    """(cos, sin) in 64 bits for positions pos [n]: [n, rope_dim/2] each."""
    f, m = _frequencies(rope_dim, scaling)
    th = pos.double()[:, None] * f
    return torch.cos(th) * m, torch.sin(th) * m


def _table(n_pos, rope_dim, scaling):
    c, s = _cos_sin(torch.arange(n_pos, device="cuda"), rope_dim, scaling)
    return torch.stack([c.float(), s.float()], -1).contiguous()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _batch(c, seed):
    """The inputs of a packed, chunks or step case."""
    g = _gen(seed)
    H, HKV = c["heads"], c["kv_heads"]
    lens = _ints(c["lens"])
    past = _ints(c["past"]) if "past" in c else [0] * len(lens)
    rows, cu = sum(lens), _starts(lens)
    s = dict(c=c, lens=lens, past=past, starts=cu, rows=rows)
    s["qkv"] = _normal(g, rows, (H + 2 * HKV) * D)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if c["kind"] == "packed":
        # the first key of a prompt draws attention from all of it
        s["qkv"][torch.tensor(cu[:-1], device="cuda"), H * D:(H + HKV) * D] *= 2.0
        return s
    bs, total = c["block"], [p + n for p, n in zip(past, lens)]
    need = [(t + bs - 1) // bs for t in total]
    common = c.get("shared", 0) // bs  # whole blocks of a common prefix, held once
    pages = common + sum(n - common for n in need)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32)
    at = common
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[:common] + order[at:at + n - common], dtype=torch.int32)
        at += n - common
    s["table"], s["max_kv"] = table.cuda(), max(total)
    s["kv_len"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    s["k"], s["v"] = _normal(g, pages * bs, HKV, D), _normal(g, pages * bs, HKV, D)
    s["q_gamma"], s["k_gamma"] = 1.0 + 0.1 * _normal(g, D), 1.0 + 0.1 * _normal(g, D)
    if c["kind"] == "step":
        s["cs"] = _table(max(total), D, "none")
        s["pos"] = torch.cat([torch.arange(p, p + n) for p, n in zip(past, lens)]).cuda()
    return s


def _rope_inputs(c, seed):
    g = _gen(seed)
    n_heads = c["heads"] + c["kv_heads"]
    x = _normal(g, c["rows"], (n_heads + c["kv_heads"]) * D)  # [Q | K | V]: V is left out
    # runs of consecutive positions, each starting anywhere
    run = max(1, c["rows"] // 8)
    r = torch.arange(c["rows"], device="cuda")
    first = torch.randint(0, c["n_pos"], ((c["rows"] + run - 1) // run,), generator=g, device="cuda")
    pos = ((first[r // run] + r % run) % c["n_pos"]).to(torch.int32)
    gamma = 1.0 + 0.1 * _normal(g, D) if c["norm"] else None
    return x, pos, gamma


def prepare(case, seed):
    c = case
    if c["kind"] == "rope":
        x, pos, gamma = _rope_inputs(c, seed)
        n_heads = c["heads"] + c["kv_heads"]
        if own:  # the table that a program makes once
            from exactinfer_amd import attention as A

            cs = A.rope_table_scaled(c["n_pos"], c["rope_dim"], THETA, A.RopeScaling(c["scaling"], FACTOR, TRAINED))
        else:
            cs = _table(c["n_pos"], c["rope_dim"], c["scaling"])
        return dict(c=c, x=x, pos=pos, gamma=gamma, cs=cs,
                    out=torch.empty((c["rows"], n_heads * D), dtype=torch.float32, device="cuda"))
    s = _batch(c, seed)
    s["out"] = torch.empty((s["rows"], c["heads"], D), dtype=torch.float32, device="cuda")
    if own:
        from exactinfer_amd import attention as A

        s["shape"] = A.AttnShape(c["heads"], c["kv_heads"])
        s["batch"] = A.PackedBatch(len(s["lens"]), s["rows"], c["heads"], c["kv_heads"])
    return s


# ------------------------------------------------------------------------------ plain forms
def _turn(x, co, si, rope_dim, layout):
    """x [rows, heads, 128] turned by co, si [rows, rope_dim/2]."""
    co, si = co[:, None], si[:, None]
    y = x.clone()
    if layout == "half":
        h = rope_dim // 2
        a, b = x[..., :h], x[..., h:rope_dim]
        y[..., :h], y[..., h:rope_dim] = a * co - b * si, a * si + b * co
    else:
        a, b = x[..., 0:rope_dim:2], x[..., 1:rope_dim:2]
        y[..., 0:rope_dim:2], y[..., 1:rope_dim:2] = a * co - b * si, a * si + b * co
    return y


def _head_norm(x, gamma):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma


def _attend(q, k, v, past, out):
    """Rows q [n, H, 128] over keys k, v [T, HKV, 128], row i seeing keys 0 .. past + i, into out [n, H, 128]."""
    n, H, _ = q.shape
    T, HKV, _ = k.shape
    G = H // HKV
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    step = max(1, min(n, BUDGET // (H * T)))
    for b in range(0, n, step):
        e = min(n, b + step)
        t = past + e
        qb = q[b:e].view(e - b, HKV, G, D).permute(1, 2, 0, 3).reshape(HKV, G * (e - b), D)
        s = torch.matmul(qb, kt[:, :, :t]) * SCALE
        s = s.view(HKV, G, e - b, t)
        rows = past + torch.arange(b, e, device=q.device)
        s.masked_fill_(torch.arange(t, device=q.device)[None, :] > rows[:, None], float("-inf"))
        s -= s.amax(-1, keepdim=True)
        s.exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(HKV, G * (e - b), t), vt[:, :t]).view(HKV, G, e - b, D) / total
        out[b:e] = o.permute(2, 0, 1, 3).reshape(e - b, H, D)


def _pool_rows(s, i, n):
    t = torch.arange(n, device="cuda")
    bs = s["c"]["block"]
    return s["table"][i].long()[t // bs] * bs + t % bs


def _plain(s):
    c = s["c"]
    H, HKV = c["heads"], c["kv_heads"]
    if c["kind"] == "rope":
        x = s["x"][:, :(H + HKV) * D].reshape(c["rows"], H + HKV, D)
        if s["gamma"] is not None:
            x = _head_norm(x, s["gamma"])
        cs = s["cs"][s["pos"].long()]
        return _turn(x, cs[..., 0], cs[..., 1], c["rope_dim"], c["layout"]).view(c["rows"], (H + HKV) * D)
    x = s["qkv"].view(s["rows"], H + 2 * HKV, D)
    q, k, v, out = x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], s["out"]
    if c["kind"] == "step":
        co, si = s["cs"][s["pos"], :, 0], s["cs"][s["pos"], :, 1]
        q = _turn(_head_norm(q, s["q_gamma"]), co, si, D, "half")
        k = _turn(_head_norm(k, s["k_gamma"]), co, si, D, "half")
    for i, (n, p) in enumerate(zip(s["lens"], s["past"])):
        a, b = s["starts"][i], s["starts"][i + 1]
        if c["kind"] == "packed":
            _attend(q[a:b], k[a:b], v[a:b], 0, out[a:b])
            continue
        rows = _pool_rows(s, i, p + n)
        if c["kind"] == "step":
            s["k"][rows[p:]], s["v"][rows[p:]] = k[a:b], v[a:b]
        _attend(q[a:b], s["k"][rows], s["v"][rows], p, out[a:b])
    return {"out": out, "k": s["k"], "v": s["v"]} if c["kind"] == "step" else out


# ------------------------------------------------------------------------------ the framework's calls
def _calls(s):
    from exactinfer_amd import attention as A

    c = s["c"]
    H, HKV = c["heads"], c["kv_heads"]
    if c["kind"] == "rope":
        return A.rope_rows(s["x"], H + HKV, s["cs"], s["pos"], rope_dim=c["rope_dim"], layout=c["layout"],
                           gamma=s["gamma"], eps=EPS, out=s["out"])
    b, qkv = s["batch"], s["qkv"]
    if c["kind"] == "packed":
        b.plan(s["cu"], s["rows"], max(s["lens"]))
        return A.attn_packed(qkv[:, :H * D], qkv[:, H * D:(H + HKV) * D], qkv[:, (H + HKV) * D:], b, s["shape"],
                             out=s["out"])
    b.plan(s["cu"], s["rows"], s["max_kv"], kv_len=s["kv_len"])
    if c["kind"] == "chunks":
        return A.attn_packed_paged(qkv[:, :H * D], s["k"], s["v"], s["table"], c["block"], b, s["shape"],
                                   out=s["out"])
    out = A.packed_step_paged(qkv, s["k"], s["v"], s["table"], c["block"], b, s["shape"], s["q_gamma"], s["k_gamma"],
                              s["cs"], out=s["out"])
    return {"out": out, "k": s["k"], "v": s["v"]}


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    H, HKV = c["heads"], c["kv_heads"]
    if c["kind"] == "rope":
        values = c["rows"] * (H + HKV) * D
        table = min(c["rows"], c["n_pos"]) * c["rope_dim"] // 2 * 8
        return {"bytes": 8 * values + table + 4 * c["rows"],
                "flops": 3 * c["rows"] * (H + HKV) * c["rope_dim"] + (4 * values if c["norm"] else 0)}
    lens = _ints(c["lens"])
    past = _ints(c["past"]) if "past" in c else [0] * len(lens)
    rows, keys = sum(lens), sum(past) + sum(lens)
    if c.get("shared"):
        keys -= (len(lens) - 1) * (c["shared"] // c["block"] * c["block"])
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
    b = 2 * rows * H * D * 4 + 2 * keys * HKV * D * 4  # q and out, every visible key
    if c["kind"] == "step":
        b += 2 * rows * HKV * D * 4 + rows * D // 2 * 8  # the new keys come from the projections, and go to the pool
    return {"bytes": b, "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------------------ in 64 bits
def _rotate64(x, pos, rope_dim, scaling, layout):
    """Each pair as a complex number times m exp(i p f): x [rows, heads, 128] in 64 bits."""
    f, m = _frequencies(rope_dim, scaling)
    turn = torch.polar(torch.full((pos.numel(), f.numel()), m, dtype=torch.float64, device="cuda"),
                       pos.double()[:, None] * f)[:, None]
    head, rest = x[..., :rope_dim], x[..., rope_dim:]
    pairs = head.unflatten(-1, (2, -1)).transpose(-1, -2) if layout == "half" else head.unflatten(-1, (-1, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2).flatten(-2) if layout == "half" else z.flatten(-2)
    return torch.cat([z, rest], -1)


def _norm64(x, gamma):
    return x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * gamma.double()


def _attention64(q, k, v, past):
    """One sequence: q [n, H, 128], k and v [T, HKV, 128]; head after head, a block of rows at a time."""
    n, H, _ = q.shape
    G = H // k.shape[1]
    out = torch.empty_like(q)
    key = torch.arange(k.shape[0], device="cuda")
    for h in range(H):
        kh, vh = k[:, h // G].t().contiguous(), v[:, h // G].contiguous()
        for b in range(0, n, 1024):
            e = min(n, b + 1024)
            s = torch.matmul(q[b:e, h], kh) * SCALE
            seen = key[None] <= past + torch.arange(b, e, device="cuda")[:, None]
            w = torch.softmax(torch.where(seen, s, torch.full_like(s, float("-inf"))), -1)
            out[b:e, h] = torch.matmul(w, vh)
    return out


def exact(case, seed):
    c = case
    H, HKV = c["heads"], c["kv_heads"]
    if c["kind"] == "rope":
        x, pos, gamma = _rope_inputs(c, seed)
        x = x.double().unflatten(-1, (-1, D))[:, :H + HKV]
        if gamma is not None:
            x = _norm64(x, gamma)
        return _rotate64(x, pos, c["rope_dim"], c["scaling"], c["layout"]).flatten(1)
    s = _batch(c, seed)
    q, k, v = s["qkv"].double().unflatten(-1, (-1, D)).split([H, HKV, HKV], 1)
    outs = []
    if c["kind"] == "packed":
        for a, b in zip(s["starts"], s["starts"][1:]):
            outs.append(_attention64(q[a:b], k[a:b], v[a:b], 0))
        return torch.cat(outs)
    pool_k, pool_v = s["k"].double(), s["v"].double()
    bs = c["block"]
    for i, (n, p) in enumerate(zip(s["lens"], s["past"])):
        a, b = s["starts"][i], s["starts"][i + 1]
        where = (s["table"][i].long()[:, None] * bs + torch.arange(bs, device="cuda")).flatten()[:p + n]
        qs = q[a:b]
        if c["kind"] == "step":
            pos = torch.arange(p, p + n, device="cuda")
            qs = _rotate64(_norm64(qs, s["q_gamma"]), pos, D, "none", "half")
            pool_k[where[p:]] = _rotate64(_norm64(k[a:b], s["k_gamma"]), pos, D, "none", "half")
            pool_v[where[p:]] = v[a:b]
        outs.append(_attention64(qs, pool_k[where], pool_v[where], p))
    out = torch.cat(outs)
    return {"out": out, "k": pool_k, "v": pool_v} if c["kind"] == "step" else out
