"""GPU tests of trees of drafted tokens over the fp32 pool, of moving accepted rows, and of a run of both with the 8-bit
cache (include/ei_cache8.h), against 64 bits.  The bar of attention is the framework's (tests/parity.py)."""
import numpy as np
import pytest
import torch

from tests.cache8_plain import D, Batch, attend64, cached64, fill_cache, i32, sees, words_of
from tests.parity import ATTN_RTOL, rel_err

pytestmark = pytest.mark.gpu


def _normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _pool64(pool, table_row, n, bs):
    t = np.arange(n)
    return pool[torch.tensor(table_row[t // bs].astype(np.int64) * bs + t % bs)].double()


def _check(b, kc, vc, q, out, bits, bar=ATTN_RTOL):
    for s, (n, total) in enumerate(zip(b.lens, b.totals)):
        if n == 0:
            continue
        r = b.rows_of(s)
        k, v = (_pool64(x, b.table_np[s], max(total, 0), b.bs) for x in (kc, vc))
        want = attend64(q[r].view(n, b.H, D).double(), k, v, sees(n, total, bits[r]))
        e = rel_err(out[r].cpu(), want.cpu())
        assert e < bar, (s, n, total, e)


CASES = [  # H, HKV, lens, past, block
    (16, 8, [1], [0], 32),
    (16, 8, [2, 1, 2], [63, 31, 500], 32),
    (8, 8, [4, 3], [100, 0], 64),
    (32, 8, [4, 5, 1], [1000, 31, 64], 64),
    (40, 8, [4, 7, 0, 3], [90, 300, 5, 2], 32),
    (16, 8, [13, 7, 13, 9], [1000, 333, 64, 2047], 32),
    (32, 8, [48, 64, 33], [700, 31, 1], 64),
    (64, 8, [100, 16], [300, 95], 128),
    (12, 4, [200, 65], [0, 77], 64),
    (8, 1, [130], [1000], 256),
]


@pytest.mark.parametrize("H,HKV,lens,past,bs", CASES)
def test_tree_attention(gpu, H, HKV, lens, past, bs):
    A = gpu
    b = Batch(A, H, HKV, lens, [p + n for p, n in zip(past, lens)], bs, seed=1, extra=2)
    kc, vc = _normal(2, b.n_blocks * bs, HKV, D), _normal(3, b.n_blocks * bs, HKV, D)
    q = _normal(4, b.rows, H * D + 8)[:, :H * D]
    mask, bits, _ = b.trees()
    out = torch.full((b.rows, H, D), 5.0, device="cuda")
    A.attn_tree_paged(q, kc, vc, b.table, bs, b.plan, b.shape, mask, out=out)
    _check(b, kc, vc, q, out, bits)
    assert bool((out[sum(lens):] == 5.0).all())
    # all bits set: causal attention
    chain = words_of([(1 << 64 * mask.shape[1]) - 1] * b.rows, mask.shape[1] + 1)
    got = A.attn_tree_paged(q, kc, vc, b.table, bs, b.plan, b.shape, chain)
    want = A.attn_packed_paged(q, kc, vc, b.table, bs, b.plan, b.shape)
    assert torch.equal(got[:sum(lens)], want[:sum(lens)])


@pytest.mark.parametrize("H,lens", [(2, [3, 9]), (8, [40, 70, 9])])
def test_rows_that_see_nothing(gpu, H, lens):
    totals = [lens[0], *lens[1:-1], 4]
    b = Batch(gpu, H, 2, lens, totals, 32, seed=5)
    kc, vc = _normal(6, b.n_blocks * 32, 2, D), _normal(7, b.n_blocks * 32, 2, D)
    q = _normal(8, b.rows, H * D)
    bits = [0] * lens[0] + [b.rng.getrandbits(64) & ~(1 << i) if i % 3 else 0 for n in lens[1:] for i in range(n)]
    out = gpu.attn_tree_paged(q, kc, vc, b.table, 32, b.plan, b.shape, words_of(bits, 1))
    _check(b, kc, vc, q, out, bits)
    assert bool((out[:lens[0]] == 0).all())


@pytest.mark.parametrize("H,lens,past", [(2, [3, 7], [40, 70]), (4, [60, 33], [45, 0]), (8, [150], [31])])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -3e38])
def test_what_a_row_does_not_see_never_reaches_it(gpu, H, lens, past, value):
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(gpu, H, 1, lens, totals, 32, seed=9)
    kc, vc = _normal(10, b.n_blocks * 32, 1, D), _normal(11, b.n_blocks * 32, 1, D)
    mask, bits, _ = b.trees(width=3)
    bad = {}
    for s, (n, total) in enumerate(zip(lens, totals)):
        bad[s] = {total - 1, total - n + n // 2}
        for t in list(bad[s]) + list(range(total, (total + 31) // 32 * 32)):
            at = int(b.table_np[s][t // 32]) * 32 + t % 32
            kc[at, 0, 5], vc[at, 0, 9] = value, value
    q = _normal(12, b.rows, H * D)
    out = gpu.attn_tree_paged(q, kc, vc, b.table, 32, b.plan, b.shape, mask)
    for s, (n, total) in enumerate(zip(lens, totals)):
        r = b.rows_of(s)
        seen = sees(n, total, bits[r])
        clean = ~seen[:, sorted(bad[s])].any(1)
        k, v = (_pool64(x, b.table_np[s], total, 32) for x in (kc, vc))
        want = attend64(q[r].view(n, H, D).double(), k, v, seen)
        assert bool(torch.isfinite(out[r][clean.cuda()]).all())
        if bool(clean.any()):
            assert rel_err(out[r][clean.cuda()].cpu(), want[clean.cuda()].cpu()) < ATTN_RTOL


def _raw(b, seed):
    return (_normal(seed, b.rows, (b.H + 2 * b.HKV) * D), 1 + 0.1 * _normal(seed + 1, D), 1 + 0.1 * _normal(seed + 2, D))


@pytest.mark.parametrize("H,HKV,lens,past,bs,extra", [(16, 8, [1, 13, 0, 30], [100, 31, 7, 0], 32, 2),
                                                     (40, 8, [48, 5], [300, 64], 64, 0)])
def test_step(gpu, H, HKV, lens, past, bs, extra):
    """Positions of the tree, slots of the batch: the pool gets the turned keys, the outputs are those of the parts."""
    A = gpu
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(A, H, HKV, lens, totals, bs, seed=13, extra=extra)
    qkv, qg, kg = _raw(b, 14)
    cs = A.rope_table(600)
    mask, bits, pos = b.trees()
    kc, vc = _normal(17, b.n_blocks * bs, HKV, D), _normal(18, b.n_blocks * bs, HKV, D)
    want_k, want_v = kc.clone(), vc.clone()
    out = A.tree_step_paged(qkv, kc, vc, b.table, bs, b.plan, b.shape, qg, kg, cs, pos=pos, mask=mask)
    rows = sum(lens)
    q = A.rope_rows(qkv, H, cs, pos, gamma=qg)
    k = A.rope_rows(qkv[:, H * D:], HKV, cs, pos, gamma=kg).view(-1, HKV, D)
    v = qkv[:, (H + HKV) * D:].reshape(-1, HKV, D)
    for s, (n, total) in enumerate(zip(lens, totals)):
        t = np.arange(total - n, total)
        at = torch.tensor(b.table_np[s][t // bs].astype(np.int64) * bs + t % bs)
        want_k[at], want_v[at] = k[b.rows_of(s)], v[b.rows_of(s)]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    _check(b, kc, vc, q, out, bits)
    got = A.attn_tree_paged(q, kc, vc, b.table, bs, b.plan, b.shape, mask)
    assert torch.equal(got[:rows], out[:rows])
    # neither mask nor positions: the packed step
    kc2, vc2 = kc.clone(), vc.clone()
    got = A.tree_step_paged(qkv, kc, vc, b.table, bs, b.plan, b.shape, qg, kg, cs)
    want = A.packed_step_paged(qkv, kc2, vc2, b.table, bs, b.plan, b.shape, qg, kg, cs)
    assert torch.equal(got[:rows], want[:rows]) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_positions_outside_the_table(gpu):
    A = gpu
    b = Batch(A, 4, 2, [6], [40], 32, seed=19)
    qkv, qg, kg = _raw(b, 20)
    kc, vc = _normal(23, b.n_blocks * 32, 2, D), _normal(24, b.n_blocks * 32, 2, D)
    before = kc.clone()
    pos = i32([34, -1, 36, 100, 101, 2 ** 31 - 1])
    A.tree_step_paged(qkv, kc, vc, b.table, 32, b.plan, b.shape, qg, kg, A.rope_table(101), pos=pos)
    at = torch.tensor([int(b.table_np[0][t // 32]) * 32 + t % 32 for t in range(34, 40)])
    same = (kc[at] == before[at]).flatten(1).all(1).cpu().tolist()
    assert same == [False, True, False, False, True, True]


# ------------------------------------------------------------------ the accepted path
def _keep_want(first, n, kept, n_kept):
    """Moves (from, to) in new rows, by the rule for lists."""
    out, before = [], -1
    for j in range(max(0, min(n_kept, len(kept)))):
        if kept[j] <= before or kept[j] >= n:
            break
        out.append((kept[j], j))
        before = kept[j]
    return out


KEPT = [  # lens, past, kept, n_kept
    ([5], [0], [[0, 2, 4]], [3]),
    ([13, 7, 1, 9], [100, 31, 500, 0], [[1, 5, 12], [0, 1, 2], [0, 0, 0], [8, 0, 0]], [3, 3, 1, 1]),
    ([20, 6, 6, 6, 0, 4], [63, 2, 2, 2, 9, 5],
     [[3, 4, 10, 19], [0, 2, 2, 3], [0, 7, 3, 4], [-1, 1, 2, 3], [0, 1, 2, 3], [1, 2, 3, 9]], [4, 4, 4, 4, 4, 9]),
    ([100], [31], [list(range(1, 98))], [97]),
    ([70, 70], [1000, 40], [list(range(0, 66)), [69] + [0] * 65], [0, -3]),
    ([8], [-3], [[2, 3, 5, 7]], [4]),
]


@pytest.mark.parametrize("lens,past,kept,n_kept", KEPT)
@pytest.mark.parametrize("kind", ["f32", "e4m3", "int8"])
def test_keep(gpu, kind, lens, past, kept, n_kept):
    A, HKV, bs = gpu, 3, 32
    totals = [p + n for p, n in zip(past, lens)]
    b = Batch(A, 6, HKV, lens, totals, bs, seed=25)
    if kind == "f32":
        pools = [_normal(26, b.n_blocks * bs, HKV, D), _normal(27, b.n_blocks * bs, HKV, D)]
        views = [p.view(b.n_blocks, bs, -1) for p in pools]
    else:
        cache = fill_cache(A, kind, b.n_blocks, bs, HKV, 28)
        views = [x.view(torch.int8).transpose(1, 2) for x in (cache.k, cache.v)] + \
            [x.transpose(1, 2) for x in (cache.k_scale, cache.v_scale)]
    want = [v.clone() for v in views]
    lengths = []
    for s, (n, total) in enumerate(zip(lens, totals)):
        first = total - n if total > 0 else -n
        moves = _keep_want(first, n, kept[s], n_kept[s])
        lengths.append(max(first + len(moves), 0))
        for x in want:
            old = x.clone()
            for src, dst in moves:
                if first + src >= 0 and first + dst >= 0:
                    f, t = first + src, first + dst
                    x[int(b.table_np[s][t // bs]), t % bs] = old[int(b.table_np[s][f // bs]), f % bs]
    if kind == "f32":
        got = A.cache_keep(*pools, b.table, bs, b.plan, b.shape, i32(kept), i32(n_kept))
    else:
        got = A.cache8_keep(cache, b.table, b.plan, i32(kept), i32(n_kept), out=b.kv_len)
        assert got.data_ptr() == b.kv_len.data_ptr()
    assert got.tolist() == lengths
    assert all(torch.equal(x, y) for x, y in zip(views, want))


def test_keep_with_missing_pages(gpu):
    """Rows that come from or go to a page that is not there stay."""
    A, bs = gpu, 32
    b = Batch(A, 2, 1, [60], [70], bs, seed=29)
    kc, vc = _normal(30, b.n_blocks * bs, 1, D), _normal(31, b.n_blocks * bs, 1, D)
    table = b.table_np.copy()
    table[0, 2] = -1  # slots from 64 on
    old = kc.clone()
    kept = [3, 30, 55, 58]
    A.cache_keep(kc, vc, i32(table), bs, b.plan, b.shape, i32([kept]), i32([4]))
    at = [int(table[0][t // bs]) * bs + t % bs for t in range(64)]
    want = old.clone()
    want[at[10]], want[at[11]] = old[at[13]], old[at[40]]
    assert torch.equal(kc, want)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind", ["f32", "e4m3", "int8"])
def test_drafting_gives_what_single_tokens_give(gpu, kind):
    """Rounds of: a tree of drafts in one step, one path of it kept.  The cache then holds what appending the kept tokens
    one by one gives, bit for bit, and their outputs agree to the bar of attention."""
    A, H, HKV, bs, n_seq = gpu, 8, 2, 32, 3
    cs = A.rope_table(512)
    qg, kg = 1 + 0.1 * _normal(40, D), 1 + 0.1 * _normal(41, D)
    table = i32(np.random.default_rng(42).permutation(3 * 6).reshape(3, 6))
    shape = A.AttnShape(H, HKV)

    def pools():
        if kind == "f32":
            return torch.zeros((18 * bs, HKV, D), device="cuda"), torch.zeros((18 * bs, HKV, D), device="cuda")
        return A.Cache8(18, bs, HKV, kind)

    def step(pool, plan, qkv, pos=None, mask=None):
        if kind == "f32":
            return A.tree_step_paged(qkv, *pool, table, bs, plan, shape, qg, kg, cs, pos=pos, mask=mask)
        return A.packed_step_cache8(qkv, pool, table, plan, shape, qg, kg, cs, pos=pos, mask=mask)

    one, two = pools(), pools()
    lens = [40, 31, 1]
    total = sum(lens)
    plan = A.PackedBatch(n_seq, 128, H, HKV)
    prompt = _normal(43, total, (H + 2 * HKV) * D)
    kv_len = i32(lens)
    plan.plan(i32(np.concatenate([[0], np.cumsum(lens)])), total, 180, kv_len=kv_len)
    for pool in (one, two):
        step(pool, plan, prompt)
    length = list(lens)
    import random
    rng = random.Random(44)
    for turn in range(6):
        n = [rng.randrange(1, 25) for _ in range(n_seq)]
        b = Batch.__new__(Batch)
        b.lens, b.totals, b.rng, b.rows = n, [x + m for x, m in zip(length, n)], rng, sum(n)
        mask, bits, pos = Batch.trees(b, width=6)
        starts = np.concatenate([[0], np.cumsum(n)])
        qkv = _normal(100 + turn, sum(n), (H + 2 * HKV) * D)
        kv_len = i32(b.totals)
        plan.plan(i32(starts), sum(n), 180, kv_len=kv_len)
        out = step(one, plan, qkv, pos=pos, mask=mask)
        # one path of each tree: the ancestors of some token
        kept = []
        for s in range(n_seq):
            leaf = rng.randrange(n[s])
            path = [i for i in range(n[s]) if bits[starts[s] + leaf] >> i & 1]
            kept.append(path[:rng.randrange(len(path) + 1)])
        most = max(max(len(k) for k in kept), 1)
        args = (i32([k + [0] * (most - len(k)) for k in kept]), i32([len(k) for k in kept]))
        if kind == "f32":
            got = A.cache_keep(*one, table, bs, plan, shape, *args, out=kv_len)
        else:
            got = A.cache8_keep(one, table, plan, *args, out=kv_len)
        assert got.tolist() == [x + len(k) for x, k in zip(length, kept)]
        single = A.PackedBatch(1, 1, H, HKV)
        for s in range(n_seq):
            for i in kept[s]:
                row = int(starts[s]) + i
                length[s] += 1
                only = i32([0] * s + [0] + [1] * (n_seq - s))
                single = A.PackedBatch(n_seq, 1, H, HKV)
                single.plan(only, 1, 180, kv_len=i32(length))
                want = step(two, single, qkv[row:row + 1])
                assert rel_err(out[row].cpu(), want[0].cpu()) < 2 * ATTN_RTOL
        for s in range(n_seq):  # what the sequences now hold
            t = torch.arange(length[s])
            pg = table[s].cpu()[t // bs].long()
            if kind == "f32":
                at = pg * bs + t % bs
                assert all(torch.equal(x[at], y[at]) for x, y in zip(one, two))
            else:
                for x, y in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
                    assert torch.equal(x.view(torch.int8)[pg, :, t % bs] if x.dim() == 4 else x[pg, :, t % bs],
                                       y.view(torch.int8)[pg, :, t % bs] if y.dim() == 4 else y[pg, :, t % bs])


@pytest.mark.parametrize("kind", ["f32", "int8"])
def test_captured_round_of_drafting(gpu, kind):
    """Plan, tree step and keep in one graph on a side stream, replayed with other lengths, trees and accepted paths,
    the program's own work between the replays; every replay against the same calls made eagerly on another pool."""
    A, H, HKV, bs, n_seq, n = gpu, 8, 2, 32, 3, 12
    b = Batch(A, H, HKV, [n] * n_seq, [200, 90, 44], bs, seed=70)
    cs, qg, kg = A.rope_table(256), 1 + 0.1 * _normal(71, D), 1 + 0.1 * _normal(72, D)

    def pool():
        if kind == "f32":
            return _normal(73, b.n_blocks * bs, HKV, D), _normal(74, b.n_blocks * bs, HKV, D)
        return fill_cache(A, kind, b.n_blocks, bs, HKV, 75)

    def tensors(p):
        return p if kind == "f32" else (p.k, p.v, p.k_scale, p.v_scale)

    cu_rows, new_len = i32(b.starts), torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    qkv = _normal(76, b.rows, (H + 2 * HKV) * D)
    mask, _, pos = b.trees()
    kept, n_kept = i32([[0] * 4] * n_seq), i32([1] * n_seq)

    def calls(p, out, lengths):
        b.plan.plan(cu_rows, b.rows, 210, kv_len=b.kv_len)
        if kind == "f32":
            A.tree_step_paged(qkv, *p, b.table, bs, b.plan, b.shape, qg, kg, cs, pos=pos, mask=mask, out=out)
            return A.cache_keep(*p, b.table, bs, b.plan, b.shape, kept, n_kept, out=lengths)
        A.packed_step_cache8(qkv, p, b.table, b.plan, b.shape, qg, kg, cs, pos=pos, mask=mask, out=out)
        return A.cache8_keep(p, b.table, b.plan, kept, n_kept, out=lengths)

    one, two = pool(), pool()
    out, stream, graph = torch.zeros((b.rows, H, D), device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        calls(pool(), out, new_len)  # (the first call, outside the capture, on a pool of its own)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            calls(one, out, new_len)
    torch.cuda.current_stream().wait_stream(stream)
    for turn, (totals, keep) in enumerate([([200, 90, 44], [[0, 3, 7, 9], [1, 2, 0, 0], [5, 0, 0, 0]]),
                                           ([130, 91, 12], [[0, 1, 2, 3], [11, 0, 0, 0], [2, 2, 2, 2]]),
                                           ([209, 40, 100], [[4, 8, 10, 11], [0, 5, 6, 20], [0, 0, 0, 0]])]):
        b.totals = totals
        new_mask, _, new_pos = b.trees()
        mask.copy_(new_mask), pos.copy_(new_pos), b.kv_len.copy_(i32(totals))
        kept.copy_(i32(keep)), n_kept.copy_(i32([4, 2 - turn % 2, turn]))
        qkv.copy_(_normal(80 + turn, *qkv.shape))
        graph.replay()
        torch.cuda.synchronize()
        want, lengths = torch.zeros_like(out), torch.zeros_like(new_len)
        calls(two, want, lengths)
        assert torch.equal(out, want) and torch.equal(new_len, lengths)
        for x, y in zip(tensors(one), tensors(two)):
            assert torch.equal(x.view(torch.int8), y.view(torch.int8))
