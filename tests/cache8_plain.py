"""Plain forms in 64 bits of what include/ei_cache8.h describes, and batches to test it with (any device)."""
import math
import random

import numpy as np
import torch

D = 128
SCALE = 1.0 / math.sqrt(D)
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def i32(a, device="cuda"):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=device)


def cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def random_tree(rng, n, width=10):
    """Ancestor bits of n tokens (own bit set), parents before children, and their depths."""
    bits, depth = [], []
    for i in range(n):
        parent = rng.randrange(max(-1, i - width), i) if i else -1
        bits.append((1 << i) | (bits[parent] if parent >= 0 else 0))
        depth.append(depth[parent] + 1 if parent >= 0 else 0)
    return bits, depth


def words_of(rows, words, device="cuda"):
    """Python integers as int64 words [rows, words]."""
    out = np.zeros((len(rows), words), np.uint64)
    for b, bits in enumerate(rows):
        for w in range(words):
            out[b, w] = (bits >> (64 * w)) & (2 ** 64 - 1)
    return torch.tensor(out.view(np.int64), device=device)


def sees(n, total, bits=None):
    """[n, total] truth values: which of a sequence's keys its n new rows see (bits: one integer a row)."""
    first = total - n
    out = torch.zeros((n, max(total, 0)), dtype=torch.bool)
    for i in range(n):
        out[i, :max(first, 0)] = True
        for j in range(i + 1):
            if first + j >= 0 and (bits is None or bits[i] >> j & 1):
                out[i, first + j] = True
    return out


def attend64(q, k, v, seen, scale=SCALE):
    """q [n, H, 128] over k, v [T, HKV, 128], all in 64 bits; keys that are not seen count for nothing, whatever they
    hold; a row without any gets zeros."""
    n, H, _ = q.shape
    HKV = k.shape[1]
    out = torch.zeros_like(q)
    for i in range(n):
        at = seen[i].nonzero()[:, 0].to(q.device)
        if at.numel() == 0:
            continue
        for h in range(HKV):
            g = slice(h * (H // HKV), (h + 1) * (H // HKV))
            w = torch.softmax(q[i, g] @ k[at, h].t().contiguous() * scale, -1)
            out[i, g] = w @ v[at, h]
    return out


def score_term64(q, k, v, seen, scale=SCALE):
    """What an output may be off by because its scores, whatever is summed how, are 32-bit numbers: a score s (log2 units)
    is rounded at least twice at its own size (its product with the key's scale, its difference to the reference),
    2^-23 |s| together, a weight then off by ln 2 times that relative to itself, numerator and denominator each
    by as much of sum w |v| / sum w."""
    n, H, _ = q.shape
    G = H // k.shape[1]
    out = attend64(q, k, v.abs(), seen, scale)
    for i in range(n):
        at = seen[i].nonzero()[:, 0].to(q.device)
        for h in range(H if at.numel() else 0):
            most = (k[at, h // G] @ q[i, h]).abs().max() * abs(scale) / math.log(2.0)
            out[i, h] *= 2 * math.log(2.0) * 2.0 ** -23 * most
    return out


def near(got, want, term, bar=1e-5):
    """The largest error against `bar` of max(|element|, rms of its head's output), the scores' term taken off; 1: at it."""
    den = torch.maximum(want.abs(), want.pow(2).mean(-1, keepdim=True).sqrt())
    off = ((got.double() - want).abs() - term).clamp(min=0.0)
    return float((off / torch.where(den == 0, torch.ones_like(den), den)).max()) / bar


def pages(rng, totals, bs, spare=3):
    """A shuffled block table for sequences of these lengths, and the number of blocks of the pool."""
    need = [max((t + bs - 1) // bs, 0) for t in totals]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    table, at = np.full((len(totals), max(max(need), 1)), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def fill_cache(A, kind, n_blocks, bs, HKV, seed, spread=1.0):
    """A Cache8 of random codes and of scales spread by 2^(spread N(0,1))."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = A.Cache8(n_blocks, bs, HKV, kind)
    for codes, scale, unit in ((c.k, c.k_scale, 1.0), (c.v, c.v_scale, 1.0)):
        x = torch.randn(codes.shape, generator=g, device="cuda")
        a = x.abs().amax(-1, keepdim=True)
        y = x / a * TOP[kind]
        codes.copy_(y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn))
        scale.copy_(unit * a[..., 0] / TOP[kind] * torch.exp2(spread * torch.randn(scale.shape, generator=g, device="cuda")))
    return c


def cached64(cache, table_row, n):
    """The first n keys and values of a sequence in 64 bits, [n, HKV, 128]; pages that are not there are zeros."""
    bs, out = cache.block_size, []
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.zeros((n, cache.n_head_kv, D), dtype=torch.float64, device=codes.device)
        for t0 in range(0, n, bs):
            blk = t0 // bs
            pg = int(table_row[blk]) if blk < len(table_row) else -1
            if 0 <= pg < cache.n_blocks:
                m = min(bs, n - t0)
                x[t0:t0 + m] = (codes[pg, :, :m].double() * scale[pg, :, :m].double()[..., None]).transpose(0, 1)
        out.append(x)
    return out


def quantised(y, kind):
    """Codes (in 64 bits) and scales of head rows y [..., 128] in fp32, by the format's operations."""
    a = y.abs().amax(-1)
    s = (a.double() / TOP[kind]).float()
    by = (TOP[kind] / a.double()).float()
    nothing, bad = a < 2.0 ** -110, ~torch.isfinite(a)
    s = torch.where(bad, torch.full_like(s, math.nan), torch.where(nothing, torch.zeros_like(s), s))
    by = torch.where(nothing | bad, torch.zeros_like(by), by)
    x = torch.where(bad[..., None], torch.zeros_like(y), y) * by[..., None]
    return (x.round() if kind == "int8" else x.to(torch.float8_e4m3fn)).double(), s


class Batch:
    """A batch of sequences with `lens` new rows and `totals` keys, its pages and its plan."""

    def __init__(self, A, H, HKV, lens, totals, bs, seed=0, extra=0, max_kv=None, spare=3):
        self.rng = random.Random(seed)
        self.A, self.H, self.HKV, self.lens, self.totals, self.bs = A, H, HKV, lens, totals, bs
        self.rows, self.starts = sum(lens) + extra, cu(lens)
        self.shape = A.AttnShape(H, HKV)
        self.table_np, self.n_blocks = pages(self.rng, totals, bs, spare)
        self.table = i32(self.table_np)
        self.kv_len = i32(totals)
        self.plan = A.PackedBatch(len(lens), self.rows, H, HKV)
        self.plan.plan(i32(self.starts), self.rows, max(max(totals), 0) if max_kv is None else max_kv,
                       kv_len=self.kv_len)

    def trees(self, width=10, extra_words=0):
        """One random tree per sequence: mask, bits by row, positions."""
        words = max(1, (max(self.lens) + 63) // 64) + extra_words
        bits, pos = [], []
        for n, total in zip(self.lens, self.totals):
            b, d = random_tree(self.rng, n, width)
            bits += b
            pos += [total - n + x for x in d]
        pad = self.rows - len(bits)
        return words_of(bits + [0] * pad, words), bits, i32(pos + [0] * pad)

    def rows_of(self, s):
        return slice(int(self.starts[s]), int(self.starts[s + 1]))
