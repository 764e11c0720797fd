"""GPU tests of the 8-bit paged cache (include/ei_cache8.h): storing, reading back and attention over it, against
64 bits.

Bars.  Codes and scales: equal to those that the format's operations in their order give (each rounded once), and
against 64 bits the code is within half a step and what the 32-bit norm and rotation are off by, some six roundings of
2^-24.  Attention: the framework's bar for fp32 attention, 1e-5 of max(|element|, rms of its head's output): q and the
weights keep 22 bits each (2^-22 of a product, with random signs over 128 of them or over the keys), everything else is
rounded as in fp32 attention.  Scales here are spread over some 2^8, so that scores reach far beyond the usual: what
their own size costs in 32 bits comes on top (score_term64).
"""
import numpy as np
import pytest
import torch

from tests.cache8_plain import (D, DTYPE, SCALE, TOP, Batch, attend64, cached64, fill_cache, i32, near, quantised,
                                score_term64, sees, words_of)
from tests.parity import ATTN_RTOL, rel_err

pytestmark = pytest.mark.gpu
KINDS = ["e4m3", "int8"]


def _normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _table64(n_pos, rope_dim, theta=1e6):
    f = theta ** (-torch.arange(rope_dim // 2, dtype=torch.float64, device="cuda") * 2 / rope_dim)
    th = torch.arange(n_pos, device="cuda").double()[:, None] * f
    return torch.cos(th), torch.sin(th)


def _turned64(x, gamma, pos, rope_dim, n_pos, eps=1e-6):
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    co, si = (t[pos.long()][:, None] for t in _table64(n_pos, rope_dim))
    h = rope_dim // 2
    a, b = x[..., :h], x[..., h:rope_dim]
    return torch.cat([a * co - b * si, a * si + b * co, x[..., rope_dim:]], -1)


# ------------------------------------------------------------------ storing
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HKV,lens,past,bs,rope_dim,extra,turned", [
    (16, 8, [1], [0], 32, 128, 0, False),
    (8, 8, [3, 0, 40, 1], [31, 5, 0, 1000], 32, 128, 5, False),
    (40, 8, [100, 7], [0, 64], 64, 64, 0, True),
    (6, 2, [65, 1, 2], [63, 127, 0], 64, 128, 1, True),
    (32, 8, [300], [4000], 128, 96, 0, False),
    (5, 1, [17, 3], [40, 0], 32, 36, 0, True),
    (8, 4, [9], [100], 32, 2, 1, False),
    (2, 2, [33], [31], 32, 126, 0, True),
    (3, 3, [2], [0], 32, 8, 0, False),
])
def test_store(gpu, kind, H, HKV, lens, past, bs, rope_dim, extra, turned):
    A = gpu
    b = Batch(A, H, HKV, lens, [p + n for p, n in zip(past, lens)], bs, seed=1, extra=extra)
    shape = A.AttnShape(H, HKV, rope_dim=rope_dim)
    width = (H + 2 * HKV) * D
    qkv = _normal(2, b.rows, width + 8)[:, :width]  # (rows of a wider buffer)
    qg, kg = 1 + 0.1 * _normal(3, D), 1 + 0.1 * _normal(4, D)
    n_pos = 5000
    cs = A.rope_table(n_pos, rope_dim)
    slot = torch.cat([torch.arange(p, p + n) for p, n in zip(past, lens)] + [torch.zeros(extra, dtype=torch.long)])
    pos = i32([(7 * int(t) + 3) % n_pos for t in slot]) if turned else None
    at = slot.cuda() if pos is None else pos
    cache = fill_cache(A, kind, b.n_blocks, bs, HKV, 5)
    before = [t.clone() for t in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
    out = torch.full((b.rows, H, D), 7.0, device="cuda")
    A.cache8_store(qkv, cache, b.table, b.plan, shape, qg, kg, cs, pos=pos, out=out)
    rows = sum(lens)
    x = qkv.reshape(b.rows, H + 2 * HKV, D)[:rows]
    want_q = A.rope_rows(qkv[:rows], H, cs, at[:rows].int(), rope_dim=rope_dim, gamma=qg).view(rows, H, D)
    assert torch.equal(out[:rows], want_q) and bool((out[rows:] == 7.0).all())
    y64 = _turned64(x[:, :H], qg, at[:rows], rope_dim, n_pos)
    assert rel_err(out[:rows].cpu(), y64.cpu()) < 1e-6
    k32 = A.rope_rows(qkv[:rows, H * D:], HKV, cs, at[:rows].int(), rope_dim=rope_dim, gamma=kg).view(rows, HKV, D)
    k64 = _turned64(x[:, H:H + HKV], kg, at[:rows], rope_dim, n_pos)
    page = torch.cat([torch.tensor(b.table_np[s][np.arange(p, p + n) // bs]) for s, (p, n) in enumerate(zip(past, lens))])
    page, off = page.long().cuda(), slot[:rows].cuda() % bs
    for codes, scale, y32, y64, b_codes, b_scale in (
            (cache.k, cache.k_scale, k32, k64, before[0], before[2]),
            (cache.v, cache.v_scale, x[:, H + HKV:], x[:, H + HKV:].double(), before[1], before[3])):
        got_c, got_s = codes[page, :, off].double(), scale[page, :, off]
        want_c, want_s = quantised(y32, kind)
        assert torch.equal(got_c, want_c) and torch.equal(got_s, want_s)
        a = y64.abs().amax(-1, keepdim=True)
        assert float(((got_s.double() - a[..., 0] / TOP[kind]).abs() / got_s.double()).max()) < 2.0 ** -20
        z = y64 * TOP[kind] / a
        if kind == "int8":
            half = torch.full_like(z, 0.5)
        else:  # half of 2^(exponent - 3), of 2^-9 below 2^-6
            half = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 4)
        assert bool(((got_c - z).abs() <= half * (1 + 2.0 ** -10) + TOP[kind] * 2.0 ** -20).all())
        # nothing else of the pool is written
        raw, want = codes.view(torch.int8).clone(), b_codes.clone()
        raw[page, :, off] = 0
        want[page, :, off] = 0
        assert torch.equal(raw, want)
        raw, want = scale.clone(), b_scale.clone()
        raw[page, :, off] = 0
        want[page, :, off] = 0
        assert torch.equal(raw, want)


@pytest.mark.parametrize("kind", KINDS)
def test_store_with_parameters_at_any_address(gpu, kind):
    """Gammas and the table at addresses that are not a multiple of 16 bytes."""
    A = gpu
    b = Batch(A, 6, 2, [7, 5], [20, 64], 32, seed=9)
    qkv, cs = _normal(10, b.rows, 10 * D), A.rope_table(80)
    g = [1 + 0.1 * _normal(11 + i, D) for i in range(2)]
    odd = []
    for t in (*g, cs):
        buf = torch.empty(t.numel() + 1, device="cuda")
        odd.append(buf[1:].view(t.shape).copy_(t))
    want, got = (A.Cache8(b.n_blocks, 32, 2, kind) for _ in range(2))
    q0 = A.cache8_store(qkv, want, b.table, b.plan, b.shape, *g, cs)
    q1 = A.cache8_store(qkv, got, b.table, b.plan, b.shape, *odd)
    assert torch.equal(q0, q1) and bool((q0 != 0).any())
    for x, y in ((want.k, got.k), (want.v, got.v), (want.k_scale, got.k_scale), (want.v_scale, got.v_scale)):
        assert torch.equal(x.view(torch.int8), y.view(torch.int8))


def _stored_values(A, kind, rows):
    """Value head rows [n, 128] stored as V of a batch of one head, and the cache and its batch."""
    n = rows.shape[0]
    b = Batch(A, 1, 1, [n], [n], 32, seed=3)
    qkv = torch.zeros((n, 3 * D), device="cuda")
    qkv[:, 2 * D:] = rows
    cache = A.Cache8(b.n_blocks, 32, 1, kind)
    ones = torch.ones(D, device="cuda")
    A.cache8_store(qkv, cache, b.table, b.plan, b.shape, ones, ones, A.rope_table(n))
    t = np.arange(n)
    page = torch.tensor(b.table_np[0][t // 32]).long().cuda()
    off = torch.tensor(t % 32).cuda()
    return cache, b, cache.v[page, 0, off], cache.v_scale[page, 0, off]


@pytest.mark.parametrize("kind", KINDS)
def test_store_every_code_and_border(gpu, kind):
    """Rows whose largest value is the largest code (scale 1): each value a code, halfway between two, or next to that."""
    codes = torch.arange(256, dtype=torch.uint8).view(DTYPE[kind]).double()
    codes = codes[torch.isfinite(codes) & (codes.abs() <= TOP[kind])].unique()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid]).float()
    x = torch.cat([x, torch.nextafter(x, torch.tensor(1e9)), torch.nextafter(x, torch.tensor(-1e9))])
    x = x[x.abs() <= TOP[kind]]
    x = torch.cat([x, torch.zeros((-x.numel()) % (D - 1))]).view(-1, D - 1)
    x = torch.cat([torch.full((x.shape[0], 1), TOP[kind]), x], 1).cuda()
    cache, _, got, scale = _stored_values(gpu, kind, x)
    want, want_s = quantised(x, kind)
    assert bool((want_s == 1.0).all()) and torch.equal(scale, want_s)
    assert torch.equal(got.double(), want)
    # nearest, ties to even: against 64 bits, no value is nearer to another code
    dist = (x.double().cpu().reshape(-1, 1) - codes[None]).abs().amin(1)
    assert torch.equal((got.double() - x.double()).abs().cpu().flatten(), dist)


@pytest.mark.parametrize("kind", KINDS)
def test_store_rows_out_of_the_ordinary(gpu, kind):
    x = torch.zeros((8, D), device="cuda")
    x[1] = 2.0 ** -120 * _normal(1, D)
    x[2] = 1.5 * 2.0 ** -109 * torch.sign(_normal(2, D))
    x[3] = 3.4e38 * torch.tanh(_normal(3, D))
    x[4] = _normal(4, D)
    x[4, 77] = float("inf")
    x[5, 127] = float("nan")
    x[6] = 1e-3
    x[7, 64] = -5.0
    cache, b, got, scale = _stored_values(gpu, kind, x)
    want, want_s = quantised(x, kind)
    assert torch.equal(got.double(), want)
    assert torch.equal(torch.isnan(scale), torch.tensor([0, 0, 0, 0, 1, 1, 0, 0]).bool().cuda())
    assert torch.equal(scale.nan_to_num(-1.0), want_s.nan_to_num(-1.0))
    assert bool((scale[:2] == 0).all()) and bool((got[:2].double() == 0).all())
    _, v = gpu.cache8_load(cache, b.table, b.plan)
    assert bool(torch.isnan(v[4:6]).all()) and bool(torch.isfinite(v[:4]).all()) and bool(torch.isfinite(v[6:]).all())


@pytest.mark.parametrize("kind", KINDS)
def test_store_and_load_where_there_is_no_place(gpu, kind):
    """Slots before 0, from max_kv on, past the table and on missing pages; positions outside the rotary table."""
    A, H, HKV, bs = gpu, 4, 2, 32
    #        slots -2 .. 2   60 .. 69        95 .. 99 of three pages, 100 .. from the fourth   missing page
    lens, totals = [5, 10, 40, 6], [3, 70, 135, 38]
    b = Batch(A, H, HKV, lens, totals, bs, seed=4, max_kv=130)
    table = b.table_np.copy()
    table[3, 1] = b.n_blocks  # slots 32 .. 37
    table = table[:, :4].copy()
    qkv = _normal(5, b.rows, (H + 2 * HKV) * D)
    slot = np.concatenate([np.arange(t - n, t) for t, n in zip(totals, lens)])
    pos = i32(np.where(np.arange(b.rows) % 7 == 3, 500, np.maximum(slot, 0)))
    cache = fill_cache(A, kind, b.n_blocks, bs, HKV, 6)
    raw = cache.k.view(torch.int8).clone()
    ones = torch.ones(D, device="cuda")
    q = A.cache8_store(qkv, cache, i32(table), b.plan, b.shape, ones, ones, A.rope_table(400), pos=pos)
    seq = np.repeat(np.arange(4), lens)
    inside = (slot >= 0) & (slot < 130) & (np.arange(b.rows) % 7 != 3)
    page = np.where(slot >= 0, table[seq, np.clip(slot // bs, 0, 3)], -1)
    page = np.where(slot // bs < 4, page, -1)
    there = (page >= 0) & (page < b.n_blocks)
    plain = qkv.view(b.rows, -1, D)[:, :H]
    same = (q == plain).flatten(1).all(1).cpu().numpy()
    assert np.array_equal(same[slot != 0], ~inside[slot != 0])
    changed = (cache.k.view(torch.int8) != raw).any(-1).any(1).cpu().numpy()
    want = np.zeros_like(changed)
    for p, t in zip(page[inside & there], slot[inside & there]):
        want[p, t % bs] = True
    assert np.array_equal(changed, want)
    out = tuple(torch.full((b.rows, HKV, D), 9.0, device="cuda") for _ in range(2))
    k, v = A.cache8_load(cache, i32(table), b.plan, out=out)
    for x, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        for r in range(b.rows):
            want = codes[page[r], :, slot[r] % bs].float() * scale[page[r], :, slot[r] % bs][:, None] if there[r] else \
                torch.zeros((HKV, D), device="cuda")
            assert torch.equal(x[r], want), r


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("HKV,lens,past,bs,extra", [(8, [1], [0], 32, 0), (8, [40, 0, 3], [100, 9, 0], 64, 3),
                                                   (3, [700, 33], [0, 4000], 128, 0), (1, [5], [27], 32, 2)])
def test_load(gpu, kind, HKV, lens, past, bs, extra):
    A = gpu
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(A, HKV, HKV, lens, totals, bs, seed=7, extra=extra)
    cache = fill_cache(A, kind, b.n_blocks, bs, HKV, 8)
    both = torch.full((b.rows, 2 * HKV * D + 4), 9.0, device="cuda")  # columns of one buffer
    A.cache8_load(cache, b.table, b.plan, out=(both[:, :HKV * D], both[:, HKV * D:2 * HKV * D]))
    for s, (n, total) in enumerate(zip(lens, totals)):
        k, v = cached64(cache, b.table_np[s], total)
        got = both[b.rows_of(s)]
        # one product of a code and a 32-bit scale, rounded once
        for x, y in ((k, got[:, :HKV * D]), (v, got[:, HKV * D:2 * HKV * D])):
            assert torch.equal(x[total - n:].float().flatten(1), y)
    assert bool((both[:, 2 * HKV * D:] == 9.0).all()) and bool((both[sum(lens):] == 9.0).all())
    k, v = A.cache8_load(cache, b.table, b.plan)
    assert k.shape == (b.rows, HKV, D) and torch.equal(k[:sum(lens)].flatten(1), both[:sum(lens), :HKV * D])


# ------------------------------------------------------------------ attention
def _near(got, q, k, v, seen, scale=None):
    """Error against 64 bits as a part of the bar."""
    kw = {} if scale is None else dict(scale=scale)
    return near(got, attend64(q, k, v, seen, **kw), score_term64(q, k, v, seen, **kw), ATTN_RTOL)


def _check(b, cache, q, out, mask_bits=None, scale=None, table=None):
    for s, (n, total) in enumerate(zip(b.lens, b.totals)):
        if n == 0:
            continue
        r = b.rows_of(s)
        k, v = cached64(cache, (b.table_np if table is None else table)[s], max(total, 0))
        e = _near(out[r], q[r].view(n, b.H, D).double(), k, v,
                  sees(n, total, None if mask_bits is None else mask_bits[r]), scale)
        assert e < 1, (s, n, total, e)


CASES = [  # H, HKV, lens, past, block
    (16, 8, [1], [0], 32),
    (32, 8, [1], [1999], 32),
    (8, 8, [1] * 7, [0, 31, 32, 33, 63, 100, 700], 64),
    (64, 8, [1, 1, 1], [5000, 31, 1], 128),
    (40, 8, [3, 1, 2, 7], [40, 300, 0, 1000], 32),
    (24, 8, [5] * 6, [100 * i for i in range(6)], 64),
    (56, 8, [9, 10], [95, 1], 32),
    (32, 8, [17, 33], [64, 3], 32),
    (12, 4, [64, 5, 0, 100], [33, 700, 12, 0], 64),
    (8, 1, [200], [500], 256),
    (32, 8, [300, 1, 1], [1000, 500, 37], 64),
    (6, 3, [128, 129], [0, 31], 32),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HKV,lens,past,bs", CASES)
def test_attention(gpu, kind, H, HKV, lens, past, bs):
    b = Batch(gpu, H, HKV, lens, [p + n for p, n in zip(past, lens)], bs, seed=11, extra=2)
    cache = fill_cache(gpu, kind, b.n_blocks, bs, HKV, 12)
    q = _normal(13, b.rows, H * D + 4)[:, :H * D]
    out = torch.full((b.rows, H, D), 5.0, device="cuda")
    gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, out=out)
    _check(b, cache, q, out)
    assert bool((out[sum(lens):] == 5.0).all())
    again = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape)
    assert torch.equal(again[:sum(lens)], out[:sum(lens)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HKV,lens,past,bs", CASES)
def test_tree_attention(gpu, kind, H, HKV, lens, past, bs):
    b = Batch(gpu, H, HKV, lens, [p + n for p, n in zip(past, lens)], bs, seed=14)
    cache = fill_cache(gpu, kind, b.n_blocks, bs, HKV, 15)
    q = _normal(16, b.rows, H * D)
    mask, bits, _ = b.trees()
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=mask)
    _check(b, cache, q, out, bits)
    # a chain is causal attention, whatever stands in the bits of later rows
    chain = words_of([(1 << 64 * mask.shape[1]) - 1] * b.rows, mask.shape[1])
    got = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=chain)
    assert torch.equal(got, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing(gpu, kind):
    """Empty masks, masks that lack their own row, fewer keys than rows, mask words that end before the rows do."""
    lens, totals = [5, 70, 9, 3, 40], [5, 70, 4, 0, 45]
    b = Batch(gpu, 8, 4, lens, totals, 32, seed=17)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 4, 18)
    q = _normal(19, b.rows, 8 * D)
    bits = [0] * 5 + [b.rng.getrandbits(64) & ~(1 << i) if i % 3 else 0 for i in range(70)] + \
        [b.rng.getrandbits(9) for _ in range(9)] + [7, 7, 7] + [0] * 40
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=words_of(bits, 1))
    for s in range(5):
        r = b.rows_of(s)
        k, v = cached64(cache, b.table_np[s], totals[s])
        seen = sees(lens[s], totals[s], bits[r])
        assert _near(out[r], q[r].view(-1, 8, D).double(), k, v, seen) < 1
        assert bool((out[r][~seen.any(1).cuda()] == 0).all())
    assert bool((out[:5] == 0).all()) and bool((out[b.rows_of(3)] == 0).all())
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape)  # causal: 9 rows over 4 keys, 3 over none
    _check(b, cache, q, out)
    assert bool((out[b.rows_of(2)][:5] == 0).all()) and bool((out[b.rows_of(3)] == 0).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,lens,past", [(4, [1, 6, 3], [40, 70, 0]), (4, [60, 33], [45, 0]), (8, [150], [31])])
def test_what_a_row_does_not_see_never_reaches_it(gpu, kind, H, lens, past):
    """NaN scales and NaN codes at keys past the end, and at new keys that some rows see and others do not."""
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(gpu, H, 1, lens, totals, 32, seed=20)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 1, 21)
    raw_k, raw_v = cache.k.view(torch.int8), cache.v.view(torch.int8)
    bad = {}  # the last new key of each sequence, and one in the middle
    for s, (n, total) in enumerate(zip(lens, totals)):
        bad[s] = {total - 1, total - n + n // 2}
        for t in list(bad[s]) + list(range(total, (total + 31) // 32 * 32)):
            pg = int(b.table_np[s][t // 32])
            for sc in (cache.k_scale, cache.v_scale):
                sc[pg, 0, t % 32] = float("nan") if t % 2 else float("inf")
            raw_k[pg, 0, t % 32], raw_v[pg, 0, t % 32] = 127, (-1 if t % 3 else 127)
    q = _normal(22, b.rows, H * D)
    mask, bits, _ = b.trees(width=3)
    for m, seen_bits in ((None, None), (mask, bits)):
        out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=m)
        for s, (n, total) in enumerate(zip(lens, totals)):
            r = b.rows_of(s)
            seen = sees(n, total, None if seen_bits is None else seen_bits[r])
            dirty = seen[:, sorted(bad[s])].any(1).cuda()
            k, v = cached64(cache, b.table_np[s], total)
            assert bool(torch.isnan(out[r][dirty]).all()) and bool(torch.isfinite(out[r][~dirty]).all())
            clean = ~dirty
            if bool(clean.any()):
                assert _near(out[r][clean], q[r].view(n, H, D).double()[clean], k, v, seen[clean.cpu()]) < 1


def test_nan_codes_alone(gpu):
    """e4m3 NaN codes under ordinary scales: only in columns, and for rows, that see them."""
    b = Batch(gpu, 4, 1, [70], [110], 32, seed=23)
    cache = fill_cache(gpu, "e4m3", b.n_blocks, 32, 1, 24)
    raw = cache.v.view(torch.int8)
    at = {45: [0, 77], 71: [5], 108: [127, 64]}
    for t, cols in at.items():
        for c in cols:
            raw[int(b.table_np[0][t // 32]), 0, t % 32, c] = 127 if c % 2 else -1
    q = _normal(25, b.rows, 4 * D)
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape)
    k, v = cached64(cache, b.table_np[0], 110)
    for i in range(70):
        clean = [c for c in range(D) if not any(c in cols and t <= 40 + i for t, cols in at.items())]
        assert bool(torch.isfinite(out[i][:, clean]).all())
        for t, cols in at.items():
            if t <= 40 + i:
                assert bool(torch.isnan(out[i][:, cols]).all())
        seen = sees(70, 110)[i:i + 1]
        q64, v64 = q[i:i + 1].view(1, 4, D).double(), v.nan_to_num(0.0)
        want = attend64(q64, k, v64, seen)
        got = torch.where(torch.isnan(out[i:i + 1]), want, out[i:i + 1].double())
        assert near(got, want, score_term64(q64, k, v64, seen), ATTN_RTOL) < 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", [([1, 3], [900, 300]), ([140], [500])])
def test_uneven_scales(gpu, kind, lens, past):
    """Values' scales over 2^80, a huge one behind a key that has no weight, huge queries against tiny keys; the output
    keeps its bits relative to what is in it."""
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(gpu, 4, 1, lens, totals, 32, seed=26)
    g = torch.Generator(device="cuda").manual_seed(27)
    base = fill_cache(gpu, kind, b.n_blocks, 32, 1, 28)
    q = _normal(29, b.rows, 4 * D)
    for name in ("wide", "falling", "rising", "behind nothing", "huge q"):
        cache = gpu.Cache8.of(base.k, base.v, base.k_scale.clone(), base.v_scale.clone())
        qq = q
        t = torch.arange(32, device="cuda").float()
        if name == "wide":
            cache.v_scale.mul_(torch.exp2(40 * torch.randn(cache.v_scale.shape, generator=g, device="cuda").clamp(-1, 1)))
        if name == "falling":
            cache.v_scale.mul_(torch.exp2(60 - 3 * t))
        if name == "rising":
            cache.v_scale.mul_(torch.exp2(3 * t - 60))
        if name == "behind nothing":  # the first key has no weight beside a strong one, and a huge value
            cache.k_scale.mul_(30.0)
            cache.v_scale[:, :, 0] *= 2.0 ** 70
            cache.k_scale[:, :, 0] = 0.0
        if name == "huge q":
            qq = q * 2.0 ** 90
            cache.k_scale.mul_(2.0 ** -90)
        out = gpu.attn_packed_cache8(qq, cache, b.table, b.plan, b.shape)
        for s, (n, total) in enumerate(zip(lens, totals)):
            r = b.rows_of(s)
            k, v = cached64(cache, b.table_np[s], total)
            seen = sees(n, total)
            want = attend64(qq[r].view(n, 4, D).double(), k, v, seen)
            # against the sum of weights times magnitudes, since values of both signs and any size cancel; a weight is
            # off by what its score is, 2^-20 of scores of up to 30 * 40 and 2^-20 besides
            size = attend64(qq[r].view(n, 4, D).double(), k, v.abs(), seen)
            bar = 2.0 ** -20 * (1 + (1200 if name == "behind nothing" else 40))
            # and a weight 2^-126 of the largest is below fp32's normal numbers: it counts as zero
            least = total * 2.0 ** -126 * v.abs().max()
            # and each weight times scale keeps 2^-25 of 2^14 to 2^15, in which the row's largest lies: times codes,
            # 2^-39 of that key's largest value, which another column's values may be far below
            most = attend64(qq[r].view(n, 4, D).double(), k, v.abs().amax(-1, keepdim=True).expand_as(v), seen)
            least = least + total * 2.0 ** -39 * most
            assert float((((out[r] - want).abs() - least).clamp(min=0.0) / size).max()) < bar, name


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", [([1, 4], [900, 300]), ([140], [500])])
@pytest.mark.parametrize("low,high", [(-80, 60), (-90, -90), (60, -80), (100, 100), (-90, 0)])
def test_scales_that_jump(gpu, kind, lens, past, low, high):
    """Values' scales of 2^low in even pages and 2^high in odd ones: small outputs keep their bits, large ones do not
    overflow on the way.  (Keys that see only the small ones are judged by them.)"""
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(gpu, 4, 1, lens, totals, 32, seed=61)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 1, 62, spread=0.3)
    for s, total in enumerate(totals):
        for i in range((total + 31) // 32):
            cache.v_scale[int(b.table_np[s][i])] *= 2.0 ** (low if i % 2 == 0 else high)
    q = _normal(63, b.rows, 4 * D)
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape)
    for s, (n, total) in enumerate(zip(lens, totals)):
        r = b.rows_of(s)
        k, v = cached64(cache, b.table_np[s], total)
        seen, q64 = sees(n, total), q[r].view(n, 4, D).double()
        want, size = attend64(q64, k, v, seen), attend64(q64, k, v.abs(), seen)
        # scores of up to 50 log2 units, and 2^-39 of a row's largest weight times scale (see test_uneven_scales)
        most = attend64(q64, k, v.abs().amax(-1, keepdim=True).expand_as(v), seen)
        off = (out[r] - want).abs() - total * 2.0 ** -39 * most
        assert float((off.clamp(min=0.0) / size).max()) < 2.0 ** -20 * 50


@pytest.mark.parametrize("kind", KINDS)
def test_missing_pages_count_as_zeros(gpu, kind):
    lens, totals = [1, 40], [200, 150]
    b = Batch(gpu, 8, 2, lens, totals, 32, seed=30)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 2, 31)
    q = _normal(32, b.rows, 8 * D)
    table = b.table_np[:, :5].copy()  # the first sequence's keys from 160 on are past the table
    table[0, 1], table[1, 2], table[1, 0] = -1, b.n_blocks, 2 ** 31 - 1
    out = gpu.attn_packed_cache8(q, cache, i32(table), b.plan, b.shape)
    _check(b, cache, q, out, table=table)


@pytest.mark.parametrize("kind", KINDS)
def test_negative_and_other_scales(gpu, kind):
    b = Batch(gpu, 8, 2, [3, 50], [130, 90], 32, seed=33)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 2, 34)
    q = _normal(35, b.rows, 8 * D)
    for scale in (-0.05, 0.0, 0.3):
        out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, scale=scale)
        _check(b, cache, q, out, scale=scale)


def test_pool_past_32_bits(gpu):
    """Codes beyond 4 GiB of the pool."""
    HKV, bs, n_blocks = 8, 128, 36000  # 4.7 GB of keys and of values
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("not enough memory")
    codes = [torch.empty((n_blocks, HKV, bs, D), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty((n_blocks, HKV, bs), device="cuda") for _ in range(2)]
    cache = gpu.Cache8.of(*codes, *scales)
    b = Batch(gpu, 16, HKV, [3, 40], [300, 129], bs, seed=36)
    table = np.array([[n_blocks - 1, 3, n_blocks - 2], [n_blocks - 3, n_blocks - 4, 0]], np.int32)
    small = fill_cache(gpu, "int8", 6, bs, HKV, 37)
    for i, pg in enumerate(table.flatten()):
        for big, x in zip((*codes, *scales), (small.k, small.v, small.k_scale, small.v_scale)):
            big[int(pg)] = x[i]
    q = _normal(38, b.rows, 16 * D)
    out = gpu.attn_packed_cache8(q, cache, i32(table), b.plan, b.shape)
    _check(b, cache, q, out, table=table)
    qkv = _normal(39, b.rows, 32 * D)
    ones = torch.ones(D, device="cuda")
    gpu.cache8_store(qkv, cache, i32(table), b.plan, b.shape, ones, ones, gpu.rope_table(300))
    k, v = gpu.cache8_load(cache, i32(table), b.plan)
    want, s = quantised(qkv[:, 24 * D:].reshape(b.rows, 8, D), "int8")
    assert torch.equal(v, (want * s.double()[..., None]).float())


# ------------------------------------------------------------------ steps, streams, graphs
def _raw(b, seed):
    g = [1 + 0.1 * _normal(seed + i, D) for i in range(2)]
    return _normal(seed, b.rows, (b.H + 2 * b.HKV) * D), g[0], g[1]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tree", [False, True])
def test_step_is_store_then_attention(gpu, kind, tree):
    A = gpu
    b = Batch(A, 16, 4, [1, 40, 0, 7], [100, 50, 3, 300], 32, seed=40, extra=3)
    qkv, qg, kg = _raw(b, 41)
    cs = A.rope_table(400)
    mask, _, pos = b.trees() if tree else (None, None, None)
    one, two = (fill_cache(A, kind, b.n_blocks, 32, 4, 42) for _ in range(2))
    out = A.packed_step_cache8(qkv, one, b.table, b.plan, b.shape, qg, kg, cs, pos=pos, mask=mask)
    q = A.cache8_store(qkv, two, b.table, b.plan, b.shape, qg, kg, cs, pos=pos)
    want = A.attn_packed_cache8(q, two, b.table, b.plan, b.shape, mask=mask)
    assert torch.equal(out[:48], want[:48])
    for x, y in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        assert torch.equal(x.view(torch.int8), y.view(torch.int8))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_step_follows_its_lengths(gpu, kind):
    """Plan and step in one graph on a side stream, replayed for other lengths, tables and trees of the same batch."""
    A, H, HKV, bs = gpu, 16, 4, 32
    b = Batch(A, H, HKV, [8, 8, 8], [300, 200, 108], bs, seed=43)
    cs = A.rope_table(400)
    qkv, qg, kg = _raw(b, 44)
    cache, other = (fill_cache(A, kind, b.n_blocks, bs, HKV, 45) for _ in range(2))
    mask, bits, pos = b.trees()
    cu_rows, out = i32(b.starts), torch.zeros((24, H, D), device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()

    def step(to, into):
        b.plan.plan(cu_rows, 24, 320, kv_len=b.kv_len)
        return A.packed_step_cache8(qkv, to, b.table, b.plan, b.shape, qg, kg, cs, pos=pos, mask=mask, out=into)

    with torch.cuda.stream(stream):
        step(cache, out)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step(cache, out)
    torch.cuda.current_stream().wait_stream(stream)
    for lens, totals in (([8, 8, 8], [300, 200, 108]), ([3, 0, 8], [290, 0, 101]), ([8, 8, 8], [301, 220, 109])):
        b.kv_len.copy_(i32(totals))
        cu_rows.copy_(i32(np.concatenate([[0], np.cumsum(lens)])))
        qkv.copy_(_normal(sum(totals), 24, (H + 2 * HKV) * D))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        rows = sum(lens)
        want = step(other, torch.full_like(out, 3.0))
        assert torch.equal(out, want) and bool((out[rows:] == 3.0).all())
        assert torch.equal(cache.k.view(torch.int8), other.k.view(torch.int8))
        assert torch.equal(cache.v_scale, other.v_scale)


def test_calls_on_two_streams(gpu):
    """Two batches, each with a workspace of its own, on two streams at once over one pool."""
    A = gpu
    batches = [Batch(A, 16, 4, [1, 30], [2000, 700], 32, seed=50 + i) for i in range(2)]
    cache = fill_cache(A, "e4m3", max(b.n_blocks for b in batches), 32, 4, 52)
    qs = [_normal(53 + i, b.rows, 16 * D) for i, b in enumerate(batches)]
    want = [A.attn_packed_cache8(q, cache, b.table, b.plan, b.shape) for q, b in zip(qs, batches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [None, None]
    for i, (q, b, st) in enumerate(zip(qs, batches, streams)):
        with torch.cuda.stream(st):
            for _ in range(5):
                got[i] = A.attn_packed_cache8(q, cache, b.table, b.plan, b.shape)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_shared_prefix_and_two_heads_of_queries(gpu):
    """Two sequences over the same pages see the same keys."""
    A = gpu
    b = Batch(A, 32, 8, [1, 1], [500, 500], 64, seed=55)
    cache = fill_cache(A, "int8", b.n_blocks, 64, 8, 56)
    table = b.table_np.copy()
    table[1] = table[0]
    q = _normal(57, 1, 32 * D).expand(2, -1).contiguous()
    out = A.attn_packed_cache8(q, cache, i32(table), b.plan, b.shape)
    _check(b, cache, q, out, table=table)


def test_refusals_in_python(gpu):
    A = gpu
    b = Batch(A, 8, 4, [4], [40], 32, seed=60)
    cache = A.Cache8(b.n_blocks, 32, 4)
    q = torch.zeros((4, 8 * D), device="cuda")
    ones = torch.ones(D, device="cuda")
    with pytest.raises(ValueError, match="KV heads"):
        A.attn_packed_cache8(q, A.Cache8(2, 32, 2), b.table, b.plan, b.shape)
    with pytest.raises(ValueError, match="block_table"):
        A.attn_packed_cache8(q, cache, b.table[0], b.plan, b.shape)
    with pytest.raises(ValueError, match="mask must be"):
        A.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=torch.zeros((3, 1), dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="int64"):
        A.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=torch.zeros((4, 1), dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="q must hold"):
        A.attn_packed_cache8(q[:3], cache, b.table, b.plan, b.shape)
    with pytest.raises(ValueError, match="no plan"):
        A.cache8_load(cache, b.table, A.PackedBatch(1, 4, 8, 4))
    with pytest.raises(ValueError, match="pos must hold"):
        A.cache8_store(torch.zeros((4, 16 * D), device="cuda"), cache, b.table, b.plan, b.shape, ones, ones,
                       A.rope_table(64), pos=i32([0, 1]))
    with pytest.raises(ValueError, match="missing"):
        A.cache8_store(torch.zeros((4, 16 * D), device="cuda"), cache, b.table, b.plan, b.shape, None, ones,
                       A.rope_table(64))
    with pytest.raises(ValueError, match="GPU tensor"):
        A.attn_packed_cache8(q, A.Cache8(b.n_blocks, 32, 4, device="cpu"), b.table, b.plan, b.shape)
