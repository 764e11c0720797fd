"""GPU tests of attention over the 8-bit pool (include/ei_cache8.h) where its scales are far from 1: everything that
storing can write, from values of 2^-110 to the largest of fp32, against 64 bits.

The bar of an element, where v_t = code * scale, w_t the row's softmax weights, N the keys and S the largest score in
log2 units:

  2^-20 (2 + S) sum_t w_t |v_t|   A score is rounded at its own size at least twice (2^-23 S together) and its weight is
                                  off by ln 2 times that, numerator and denominator alike: below 2^-22 S.  Products of
                                  two operands of 22 bits, and fp32 sums over tiles, waves and parts: below 2^-19.
  2^-38 N max_t w_t scale_t max_d |code_td|
                                  Planes of a weight times scale end at half of 2^-24 where the row's largest weight
                                  times scale is 2^13 or more: 2^-38 of it for each key, times codes.
  sum of w_t |v_t| over w_t < 2^-116
                                  Such weights may count as zero.
"""
import math

import pytest
import torch

from tests.cache8_plain import D, SCALE, Batch, cached64, fill_cache, i32, sees

pytestmark = pytest.mark.gpu
KINDS = ["e4m3", "int8"]
# units of single tokens and drafts; of up to 64 and of up to 128 rows; more than one of them
BATCHES = [([1, 4], [900, 300]), ([12, 15], [400, 700]), ([35], [700]), ([140], [500])]


def _normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _worst(q, k, v, seen, got):
    """The largest error as a part of its bar (q [n, H, 128], k and v [N, 1, 128] in 64 bits)."""
    n, H, _ = q.shape
    k, v, N = k[:, 0], v[:, 0], v.shape[0]
    hidden = ~seen.to(q.device)[:, None].expand(n, H, N)
    s = (q.reshape(-1, D) @ k.t().contiguous()).view(n, H, N) * (SCALE / math.log(2.0))
    s = s.masked_fill(hidden, -math.inf)
    w = torch.softmax(s * math.log(2.0), -1)
    S = s.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True)
    def mix(w, v):
        return (w.reshape(-1, N) @ v).view(n, H, D)
    bar = 2.0 ** -20 * (2 + S) * mix(w, v.abs())
    bar = bar + 2.0 ** -38 * N * (w * v.abs().amax(-1)).amax(-1, keepdim=True)
    bar = bar + mix(torch.where(w < 2.0 ** -116, w, torch.zeros_like(w)), v.abs())
    assert bool(torch.isfinite(got).all())
    off = (got.double() - mix(w, v)).abs()
    return float((off / torch.where(bar == 0, torch.ones_like(bar), bar)).max())


def _check(b, cache, q, out, mask_bits=None):
    for s, (n, total) in enumerate(zip(b.lens, b.totals)):
        r = b.rows_of(s)
        k, v = cached64(cache, b.table_np[s], total)
        seen = sees(n, total, None if mask_bits is None else mask_bits[r])
        e = _worst(q[r].view(n, b.H, D).double(), k, v, seen, out[r])
        assert e < 1, (s, n, total, e)


def _batch(gpu, lens, past, seed):
    return Batch(gpu, 4, 1, lens, [p + n for p, n in zip(past, lens)], 32, seed=seed)


def _keys_of_ones(gpu, kind, b, seed, log2_score):
    """A cache whose keys give queries of ones the log2 scores log2_score(t) (a function of the keys' numbers)."""
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 1, seed, spread=0.2)
    cache.k.copy_(torch.ones(cache.k.shape, device="cuda").to(cache.k.dtype))
    for s, total in enumerate(b.totals):
        t = torch.arange(total, device="cuda")
        page = i32(b.table_np[s]).long()[t // 32]
        cache.k_scale[page, 0, t % 32] = log2_score(t).float() * (math.log(2.0) / SCALE / D)
    return cache


# ------------------------------------------------------------------ tiny values
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES + [([1], [20000])])
@pytest.mark.parametrize("power", [-84, -98, -104, -110])
def test_tiny_values(gpu, kind, lens, past, power):
    """Scales of 2^-9 to 2^-4 times 2^power: down to the smallest that are stored."""
    b = _batch(gpu, lens, past, 1)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 1, 2, spread=0.2)
    cache.v_scale.clamp_(2.0 ** -9, 2.0 ** -4).mul_(2.0 ** power)
    q = _normal(3, b.rows, 4 * D)
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES)
def test_tiny_values_behind_others(gpu, kind, lens, past):
    """Tiny values at the keys that have all the weight, ordinary ones at earlier keys that have next to none."""
    b = _batch(gpu, lens, past, 4)
    cache = _keys_of_ones(gpu, kind, b, 5, lambda t: torch.where(t < 200, -150.0, 0.0))
    for s, total in enumerate(b.totals):
        t = torch.arange(200, total, device="cuda")
        cache.v_scale[i32(b.table_np[s]).long()[t // 32], 0, t % 32] *= 2.0 ** -105
    q = torch.ones((b.rows, 4 * D), device="cuda")
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))


@pytest.mark.parametrize("kind", KINDS)
def test_tiny_values_as_stored(gpu, kind):
    """A step whose values are around 2^-108 gives what the same step gives for them times 2^108, scaled."""
    A = gpu
    lens, past = [3, 40, 1], [0, 0, 0]
    outs = []
    for power in (0, -108):
        b = Batch(A, 8, 4, lens, [p + n for p, n in zip(past, lens)], 32, seed=6)
        qkv = _normal(7, b.rows, 16 * D)
        qkv[:, 12 * D:] = (1 + qkv[:, 12 * D:].abs()) * 2.0 ** power
        cache, ones = A.Cache8(b.n_blocks, 32, 4, kind), torch.ones(D, device="cuda")
        outs.append(A.packed_step_cache8(qkv, cache, b.table, b.plan, b.shape, ones, ones, A.rope_table(64)))
    # The same codes, in two arithmetics: positive values, so that each is within 2^-20 (2 + S) of itself (the bar
    # above), scores of normed rows at most 128 / sqrt(128) log2(e) = 16.4 (of keys off by 1/254 or 1/16 of themselves, 17.4)
    assert bool(((outs[0] - outs[1] * 2.0 ** 108).abs() <= 2 * 2.0 ** -20 * 19.4 * outs[0]).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES)
@pytest.mark.parametrize("score,power", [(0.0, -110), (60.0, -50)])
def test_zeros_beside_tiny_values(gpu, kind, lens, past, score, power):
    """Values that are zero (and a page that is not there) with as much weight as tiny ones, or much more."""
    b = _batch(gpu, lens, past, 8)
    cache = _keys_of_ones(gpu, kind, b, 9, lambda t: torch.where(t % 5 == 2, score, 0.0))
    cache.v_scale.mul_(2.0 ** power)
    table = b.table_np.copy()
    for s, total in enumerate(b.totals):
        t = torch.arange(2, total, 5, device="cuda")
        cache.v_scale[i32(table[s]).long()[t // 32], 0, t % 32] = 0.0
        table[s, 1] = -1
    b.table_np = table
    q = torch.ones((b.rows, 4 * D), device="cuda")
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, i32(table), b.plan, b.shape))


# ------------------------------------------------------------------ scales that a row does not see
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [60, 100, 117])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("n", [4, 15, 40])
def test_huge_values_that_a_row_does_not_see(gpu, kind, power, tree, n):
    """Finite huge values at new keys that some rows see and others do not, beside scales of some 2^-20: rows that do
    not see them keep their bits.  Eight sequences of eight KV heads, so that a workgroup takes several tiles of one; nearly
    all weight is at the new keys, which share their tiles with the huge ones."""
    H, HKV, past, seqs = 32, 8, 990, 8
    total = past + n
    b = Batch(gpu, H, HKV, [n] * seqs, [total] * seqs, 32, seed=11)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, HKV, 12, spread=0.2)
    cache.k.copy_(torch.ones(cache.k.shape, device="cuda").to(cache.k.dtype))
    cache.v_scale.mul_(2.0 ** -14)
    huge = sorted({total - 1, past + n // 2})
    t = torch.arange(total, device="cuda")
    for s in range(seqs):
        page = i32(b.table_np[s]).long()[t // 32]
        score = torch.where(t < past, -30.0, 0.1 * (t % 7)).float() * (math.log(2.0) / SCALE / D)
        cache.k_scale[page, :, t % 32] = score[:, None]
        for h in huge:
            cache.v_scale[page[h], :, h % 32] = 2.0 ** power
    q = 1 + 0.1 * _normal(13, b.rows, H * D)
    mask, bits, _ = b.trees(width=3) if tree else (None, None, None)
    out = gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape, mask=mask)
    for s in range(seqs):
        r = b.rows_of(s)
        k, v = cached64(cache, b.table_np[s], total)
        seen = sees(n, total, None if bits is None else bits[r])
        for rows in (~seen[:, huge].any(1), seen[:, huge].any(1)):
            at = rows.cuda()
            if not bool(rows.any()):
                continue
            for h in (0, 5):
                heads = slice(h * (H // HKV), (h + 1) * (H // HKV))
                q64 = q[r].view(n, H, D).double()[at][:, heads]
                assert _worst(q64, k[:, h:h + 1], v[:, h:h + 1], seen[rows], out[r][at][:, heads]) < 1, (s, h)


# ------------------------------------------------------------------ huge values
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES + [([1], [20000])])
@pytest.mark.parametrize("power", [60, 100, 118])
def test_huge_values_of_one_sign(gpu, kind, lens, past, power):
    """Sums over the keys would pass fp32's range long before they are divided; the outputs do not."""
    b = _batch(gpu, lens, past, 14)
    cache = fill_cache(gpu, kind, b.n_blocks, 32, 1, 15, spread=0.2)
    cache.v.view(torch.int8).bitwise_and_(0x7F) if kind == "e4m3" else cache.v.copy_(cache.v.abs())
    cache.v_scale.fill_(2.0 ** power)
    q = _normal(16, b.rows, 4 * D)
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES + [([1], [20000])])
def test_small_weights_of_huge_values(gpu, kind, lens, past):
    """A key with nearly all the weight, and many with 2^-25 of it each."""
    b = _batch(gpu, lens, past, 17)
    cache = _keys_of_ones(gpu, kind, b, 18, lambda t: torch.where(t == 100, 25.0, 0.0))
    cache.v_scale.mul_(2.0 ** 121)
    for s in range(len(lens)):  # the values of that key are zero in half of the columns
        cache.v[int(b.table_np[s][3]), 0, 4].view(torch.int8)[:64] = 0
    q = torch.ones((b.rows, 4 * D), device="cuda")
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,past", BATCHES)
def test_huge_values_without_weight(gpu, kind, lens, past):
    """Huge values at keys that have next to no weight beside tiny ones at the others."""
    b = _batch(gpu, lens, past, 19)
    cache = _keys_of_ones(gpu, kind, b, 20, lambda t: torch.where(t % 50 == 7, -300.0, 0.0))
    for s, total in enumerate(b.totals):
        t = torch.arange(total, device="cuda")
        cache.v_scale[i32(b.table_np[s]).long()[t // 32], 0, t % 32] = \
            torch.where(t % 50 == 7, 2.0 ** 117, 2.0 ** -90 * (1 + 0.01 * (t % 32))).float()
    q = torch.ones((b.rows, 4 * D), device="cuda")
    _check(b, cache, q, gpu.attn_packed_cache8(q, cache, b.table, b.plan, b.shape))
