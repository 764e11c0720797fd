"""GPU tests of the packed batch (include/ei_packed.h): the plan's cover, attention over packed prompts and
over paged chunks, and the whole step, against softmax attention in 64 bits.

The bar is the framework's own for fp32 attention, 1e-5 of max(|element|, rms of its head's output)
(tests/parity.py): a score of 128 products is off by some 2^-21 of the sum of their sizes, a weight by as
much, and sums over T keys round at most T/16 * 6 + T/32 times at 2^-24, with random signs.
"""
import numpy as np
import pytest
import torch

from tests.parity import ATTN_RTOL, rel_err

pytestmark = pytest.mark.gpu

D = 128
SCALE = 1.0 / np.sqrt(D)


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _attend64(q, k, v, kv_len, scale=SCALE):
    """q [n, H, 128] over k, v [T, HKV, 128] (float64 tensors); row i sees keys 0 .. kv_len - n + i."""
    n, H, _ = q.shape
    T, HKV, _ = k.shape
    out = torch.zeros_like(q)
    sees = torch.arange(T, device=q.device)[None] <= (kv_len - n + torch.arange(n, device=q.device))[:, None]
    for h in range(H):
        s = q[:, h] @ k[:, h // (H // HKV)].t().contiguous() * scale
        s = torch.where(sees, s, -torch.inf)
        w = torch.softmax(s, -1)
        out[:, h] = torch.nan_to_num(w) @ v[:, h // (H // HKV)]
    out[kv_len - n + torch.arange(n, device=q.device) < 0] = 0.0
    return out


def _shares(HKV):
    return max(1, 256 // HKV)


def _read_plan(batch, lens, rows, H, HKV):
    """The plan's header and two lists, wide and few-row: their units and shares (first, first tile, last, last tile,
    last share of a merge, 3 words, the unit it starts with, the unit to merge)."""
    raw = batch.buf.cpu().numpy()
    head = raw[:256].view(np.int32)
    G, n_seq, shares = H // HKV, len(lens), 96 * _shares(HKV)
    wide = 256 + 16 * n_seq
    few = wide + 32 * (rows * G // 128 + n_seq)
    at = few + 32 * n_seq

    def units(start, n):
        return raw[start:start + 32 * n].view(np.int32).reshape(-1, 8)

    return (head, units(wide, head[7] + head[8]), raw[at:at + shares].view(np.int32).reshape(-1, 24),
            units(few, head[9]), raw[at + shares:at + 2 * shares].view(np.int32).reshape(-1, 24))


BATCHES = [  # H, HKV, lens, kv_len (None: whole prompts)
    (16, 8, [1], None), (16, 8, [37, 1, 96, 5, 64], None), (32, 8, [0, 40, 0, 0, 700, 3], None),
    (40, 8, [700, 33, 1501, 128, 2, 940], None), (8, 1, [2000], None), (8, 8, [300] * 9, None),
    (32, 8, [4096, 300, 17, 2048], None), (12, 4, [1] * 40, [1 + 97 * i for i in range(40)]),
    (16, 8, [1, 512, 1, 300, 1], [2001, 2048, 34, 300, 4101]), (32, 8, [5] * 16, [1024 + 37 * i for i in range(16)]),
    (16, 8, [4, 9, 3], [2, 0, 3]), (8, 8, [1], [30000]), (6, 3, [1000, 0, 17], [1000, 5000, 0]),
]


@pytest.mark.parametrize("H,HKV,lens,kv", BATCHES)
def test_plan_covers_every_unit_once(gpu, H, HKV, lens, kv):
    """Every unit in the deal or on the line exactly once, with its tiles; cuts in order, inside their
    units; and no workgroup more than a unit's passes over an equal share."""
    rows, G = sum(lens), H // HKV
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(_cu(lens)), rows, max(kv or lens), kv_len=None if kv is None else _i32(kv))
    head, wide, wide_shares, few, few_shares = _read_plan(b, lens, rows, H, HKV)
    N = _shares(HKV)
    want = {True: {}, False: {}}
    for s, n in enumerate(lens):
        total = n if kv is None else kv[s]
        for u in range((n * G + 127) // 128):
            last = min(n - 1, (128 * u + 127) // G)
            want[n * G - 128 * u <= 32][s, u] = (max(0, min(total, total - n + last + 1)) + 31) // 32
    rounds, dealt, line = int(head[6]), int(head[7]), int(head[8])
    assert dealt == rounds * N and dealt + line == len(wide)
    load = np.zeros(N, int)
    for is_few, units, shares, first, (once, turn) in ((False, wide, wide_shares, dealt, (5, 2)),
                                                       (True, few, few_shares, 0, (5, 8))):
        cost = want[is_few]
        assert {(int(x[4]), int(x[3])): int(x[5]) for x in units} == cost and len(units) == len(cost)
        for x in units:
            s = int(x[4])
            assert (int(x[0]), int(x[1]), int(x[2])) == (int(_cu(lens)[s]), lens[s], lens[s] if kv is None else kv[s])
        tiles = units[:, 5].astype(int)
        if first:
            assert np.all(np.diff(tiles) <= 0)  # descending
        for i in range(first):
            r, j = divmod(i, N)
            load[N - 1 - j if r % 2 else j] += tiles[i] + once
        share = -(-sum(t + once for t in cost.values()) // N)
        while turn > max(share, 1) and sum(t + 5 for c in want.values() for t in c.values()) <= 7 * N:
            turn //= 2
        n, at = len(units) - first, (0, 0)
        begins, ends = {}, {}  # shares in which a cut unit begins; the last share with a part of a unit
        for j in range(N):
            (a, ta), (e, te) = shares[j, 0:2], shares[j, 2:4]
            assert (a, ta) == at and (a, ta) <= (e, te)
            at = (e, te)
            assert te == 0 or (e < n and turn <= te <= tiles[first + e] - turn and te % turn == 0)
            for i in range(a, min(e + 1, n)):
                lo, hi = (ta if i == a else 0), (te if i == e else tiles[first + i])
                if i < e or te > 0:
                    load[j] += hi - lo + once
                    if lo == 0 and hi < tiles[first + i]:
                        begins[j] = i
                    if lo > 0:
                        ends[i] = j
            if first or a < n:
                assert np.array_equal(shares[j, 8:16], units[j if first else a])
        assert at == (n, 0)
        for j in range(N):
            assert shares[j, 4] == (ends[begins[j]] if j in begins else 0)
            if j in begins:
                assert np.array_equal(shares[j, 16:24], units[first + begins[j]])
        fair = sum(sum(t + c for t in want[f].values()) for f, c in ((False, 5), (True, 5))[:1 + is_few]) / N
        assert load.max() <= fair + 4 * once + 2 * turn + (max(tiles, default=0) if first else 0) + 24 * is_few


def _prompts(H, HKV, lens, seed, extra=0):
    rows = sum(lens) + extra
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn((rows, (H + 2 * HKV) * D), generator=g, device="cuda")
    return qkv, qkv[:, :H * D], qkv[:, H * D:(H + HKV) * D], qkv[:, (H + HKV) * D:]


def _check_prompts(out, q, k, v, lens, H, HKV, scale=SCALE):
    cu = _cu(lens)
    for s, n in enumerate(lens):
        if n == 0:
            continue
        r = slice(int(cu[s]), int(cu[s + 1]))
        ref = _attend64(q[r].double().view(n, H, D), k[r].double().view(n, HKV, D), v[r].double().view(n, HKV, D), n,
                        scale)
        e = rel_err(out[r].cpu().numpy(), ref.cpu().numpy())
        assert e <= ATTN_RTOL, (s, n, e)


@pytest.mark.parametrize("H,HKV,lens", [
    (8, 8, [1]), (16, 8, [2, 1]), (16, 8, [37, 1, 96, 5, 64]), (32, 8, [0, 40, 0, 0, 300, 3, 0]),
    (40, 8, [31, 32, 33, 64, 65, 127, 128, 129]), (18, 6, [77, 200]), (8, 1, [257, 13]), (48, 8, [50, 51]),
    (56, 8, [19, 90]), (6, 3, [100, 45]), (32, 8, [1100, 900, 17]), (8, 8, [600] * 3),
])
def test_packed_prompts(gpu, H, HKV, lens):
    qkv, q, k, v = _prompts(H, HKV, lens, 11)
    b = gpu.PackedBatch(len(lens), sum(lens), H, HKV)
    b.plan(_i32(_cu(lens)), sum(lens), max(lens))
    before = qkv.clone()
    out = gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV))
    _check_prompts(out, q, k, v, lens, H, HKV)
    assert torch.equal(qkv, before)
    # the same bits again, planned again
    b.plan(_i32(_cu(lens)), sum(lens), max(lens))
    assert torch.equal(gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV)), out)


def test_rows_behind_the_last_sequence_stay(gpu):
    H, HKV, lens = 16, 8, [40, 25]
    qkv, q, k, v = _prompts(H, HKV, lens, 12, extra=30)
    qkv[65:] = float("nan")
    b = gpu.PackedBatch(4, 200, H, HKV)
    b.plan(_i32(_cu(lens)), 95, 40)
    out = torch.full((95, H, D), 3.0, device="cuda")
    gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV), out=out)
    _check_prompts(out, q, k, v, lens, H, HKV)
    assert (out[65:] == 3.0).all()


def test_wrong_lengths_write_nothing(gpu):
    """cu_rows that fall, start below 0 or count more rows than there are; a plan of other heads."""
    H, HKV = 16, 8
    _, q, k, v = _prompts(H, HKV, [64], 13)
    for cu in ([0, 40, 30, 64], [-1, 20, 40, 64], [0, 20, 40, 65], [0, 70, 64, 64]):
        b = gpu.PackedBatch(3, 64, H, HKV)
        b.plan(_i32(cu), 64, 64)
        out = torch.full((64, H, D), 3.0, device="cuda")
        gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV), out=out)
        assert (out == 3.0).all(), cu
    b = gpu.PackedBatch(3, 64, 32, 8)
    b.plan(_i32([0, 64]), 64, 64)
    out = torch.full((64, H, D), 3.0, device="cuda")
    from exactinfer_amd import _capi
    stream = torch.cuda.current_stream().cuda_stream
    _capi.call("ei_attn_packed", stream, q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0),
               out.data_ptr(), 1, 64, H, HKV, D, 0.1, b.buf.data_ptr(), b.nbytes, b.ws.data_ptr(), b.ws_nbytes)
    assert (out == 3.0).all()
    # a plan over a cache, given to the call whose keys are the rows
    b.plan(_i32([0, 64]), 64, 200, kv_len=_i32([200]))
    out = torch.full((64, 32, D), 3.0, device="cuda")
    _, q, k, v = _prompts(32, 8, [64], 13)
    _capi.call("ei_attn_packed", stream, q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0),
               out.data_ptr(), 1, 64, 32, 8, D, 0.1, b.buf.data_ptr(), b.nbytes, b.ws.data_ptr(), b.ws_nbytes)
    assert (out == 3.0).all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 1e-30])
def test_other_scales(gpu, scale):
    H, HKV, lens = 16, 8, [70, 33]
    _, q, k, v = _prompts(H, HKV, lens, 14)
    q, k = q * 0.3, k * 0.3  # (scores of up to some 10 at scale 1)
    b = gpu.PackedBatch(2, 103, H, HKV)
    b.plan(_i32(_cu(lens)), 103, 70)
    out = gpu.attn_packed(q.contiguous(), k.contiguous(), v.contiguous(), b, gpu.AttnShape(H, HKV), scale=scale)
    _check_prompts(out, q, k, v, lens, H, HKV, scale)


@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan"), 3e38, 1e30, -1e25])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, what):
    """A key or value row of infinities, NaN or huge values: rows before it, and other sequences, have the
    outputs they have without it."""
    H, HKV, lens = 16, 8, [50, 90, 41]
    _, q, k, v = _prompts(H, HKV, lens, 15)
    shape = gpu.AttnShape(H, HKV)
    b = gpu.PackedBatch(3, sum(lens), H, HKV)
    b.plan(_i32(_cu(lens)), sum(lens), 90)
    clean = gpu.attn_packed(q, k, v, b, shape)
    bad_row = 50 + 45  # row 45 of the second sequence
    for target in ("k", "v"):
        k2, v2 = k.contiguous(), v.contiguous()
        (k2 if target == "k" else v2)[bad_row, 5::7] = what
        out = gpu.attn_packed(q, k2, v2, b, shape)
        keep = np.r_[0:bad_row, 140:181]
        e = rel_err(out[keep].cpu().numpy(), clean[keep].cpu().numpy())
        assert e <= ATTN_RTOL, (target, e)


def test_visible_infinities_and_nan(gpu):
    """A NaN value reaches the rows that see it, in its column alone; a key whose scores are -inf has weight
    zero, and its infinite score +inf makes the row NaN, as in the formula."""
    H, HKV, n = 8, 8, 80
    _, q, k, v = _prompts(H, HKV, [n], 16)
    shape = gpu.AttnShape(H, HKV)
    b = gpu.PackedBatch(1, n, H, HKV)
    b.plan(_i32([0, n]), n, n)
    clean = gpu.attn_packed(q, k, v, b, shape)
    v2 = v.contiguous()
    v2[20, 3] = float("nan")
    v2[33, 130] = float("inf")
    out = gpu.attn_packed(q, k.contiguous(), v2, b, shape)
    seen = torch.zeros_like(clean, dtype=torch.bool)
    seen[20:, 0, 3] = True
    assert torch.equal(torch.isnan(out), seen)
    assert (out[33:, 1, 2] == float("inf")).all()
    seen[33:, 1, 2] = True
    assert rel_err(torch.where(seen, clean, out).cpu().numpy(), clean.cpu().numpy()) <= ATTN_RTOL
    # keys whose scores are -inf (against positive q) in one head
    q2, k2 = q.contiguous(), k.contiguous()
    q2[:, 0] = q2[:, 0].abs() + 0.1
    k2[10, 0] = float("-inf")
    out = gpu.attn_packed(q2, k2, v.contiguous(), b, shape)
    ref = _attend64(q2.double().view(n, H, D), k2.double().view(n, HKV, D), v.double().view(n, HKV, D), n)
    assert torch.isfinite(out).all() and rel_err(out.cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL
    k2[10, 0] = float("inf")
    out = gpu.attn_packed(q2, k2, v.contiguous(), b, shape)
    assert torch.isnan(out[10:, 0]).all() and torch.isfinite(out[:10]).all() and torch.isfinite(out[:, 1:]).all()


def _run_prompts(gpu, q, k, v, lens, H, HKV, scale=None):
    b = gpu.PackedBatch(len(lens), sum(lens), H, HKV)
    b.plan(_i32(_cu(lens)), sum(lens), max(lens))
    return gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV), scale=scale)


@pytest.mark.parametrize("H,HKV,lens", [(16, 8, [100, 7, 300]), (32, 8, [4, 8, 1]), (8, 1, [60])])
@pytest.mark.parametrize("e_qk,e_v", [(60, 0), (-60, 0), (0, 100), (0, -90), (100, 30), (-30, 60)])
def test_powers_of_two_come_out_exactly(gpu, H, HKV, lens, e_qk, e_v):
    """q by 2^e and k by 2^-e change nothing, v by 2^e the output by 2^e: every scaling in the kernels is a
    power of two that follows the values."""
    _, q, k, v = _prompts(H, HKV, lens, 101)
    ref = _run_prompts(gpu, q, k, v, lens, H, HKV)
    out = _run_prompts(gpu, (q * 2.0 ** e_qk).contiguous(), (k * 2.0 ** -e_qk).contiguous(),
                       (v * 2.0 ** e_v).contiguous(), lens, H, HKV)
    assert torch.equal(out, ref * 2.0 ** e_v)


@pytest.mark.parametrize("H,HKV,lens", [(16, 8, [150, 40]), (32, 8, [8, 5])])
@pytest.mark.parametrize("what", ["k_row", "k_channel", "v_row", "v_column", "v_zero", "v_heads", "q_row"])
def test_uneven_magnitudes(gpu, H, HKV, lens, what):
    """Rows and columns far larger or smaller than the others, against 64 bits."""
    _, q, k, v = (t.contiguous() for t in _prompts(H, HKV, lens, 102))
    if what == "k_row":  # every seventh key large: its row's own scaling must not cost the others
        k[::7] *= 1000.0
        q *= 1e-3
    elif what == "k_channel":
        k[:, 5::128] *= 300.0
        q[:, 5::128] *= 1e-3
    elif what == "v_row":  # a value row 2^30 times the others, at a key whose weight is e^-40 or so
        k[3] = 0.0
        q[:, ::128] = 40.0
        k[:, ::128] = 12.0
        k[3, ::128] = 0.0
        v[3] *= 2.0 ** 30
    elif what == "v_column":
        v[:, 9::128] *= 1e-6
    elif what == "v_zero":
        v[:] = 0.0
    elif what == "v_heads":
        v[:, :D] *= 1e20
        v[:, D:2 * D] *= 1e-30
    else:
        q[11] *= 50.0
    out = _run_prompts(gpu, q, k, v, lens, H, HKV)
    if what == "v_row":
        # Scores of 40 * 12 / sqrt(128) lie near 61 in log2 units, where an fp32 sum is rounded by up to 2^-18:
        # 127 additions move a score by at most 127 * 2^-18, a weight by that times ln 2 of itself, and an
        # output by twice as much of the largest ordinary value.  (Unnoticed, the planes of V would be off by
        # 2^-25 of their range, 2^-6 here, five times that.)
        tol = 2 * 127 * 2.0 ** -18 * np.log(2) * v[np.r_[0:3, 4:v.shape[0]]].abs().max().item()
        for a, n in zip(_cu(lens), lens):
            r = slice(int(a), int(a) + n)
            ref = _attend64(q[r].double().view(n, H, D), k[r].double().view(n, HKV, D), v[r].double().view(n, HKV, D), n)
            assert (out[r] - ref).abs().max().item() <= tol
        return
    if what == "q_row":
        # A row 50 times the others has scores of hundreds of log2 units.  An fp32 sum of 128 products is off by at
        # most 127 * 2^-24 of the sum of their magnitudes, a weight by that times ln 2 of itself, and the row's output
        # by twice as much of the largest value.  The other rows keep the tolerance below.
        most = v.abs().max().item()
        for a, n in zip(_cu(lens), lens):
            a = int(a)
            if not a <= 11 < a + n:
                continue
            r = slice(a, a + n)
            ref = _attend64(q[r].double().view(n, H, D), k[r].double().view(n, HKV, D), v[r].double().view(n, HKV, D), n)
            mags = q[11].double().view(HKV, -1, D).abs() @ k[a:12].double().view(-1, HKV, D).abs().permute(1, 2, 0).contiguous()
            off = 127 * 2.0 ** -24 * mags.max().item() * SCALE * np.log2(np.e)
            assert (out[11] - ref[11 - a]).abs().max().item() <= 2 * off * np.log(2) * most
            out[11] = ref[11 - a]
    _check_prompts(out, q, k, v, lens, H, HKV)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_query_row_stays_its_own(gpu, bad):
    H, HKV, lens = 16, 8, [70, 6]
    _, q, k, v = (t.contiguous() for t in _prompts(H, HKV, lens, 103))
    clean = _run_prompts(gpu, q, k, v, lens, H, HKV)
    q[33, 4] = bad   # head 0 of a row of the wide unit
    q[72, 130] = bad  # head 1 of a row of the few-row unit
    out = _run_prompts(gpu, q, k, v, lens, H, HKV)
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[33, 0] = keep[72, 1] = False
    assert torch.isnan(out[33, 0]).all() and torch.isnan(out[72, 1]).all()
    assert rel_err(torch.where(keep, out, clean).cpu().numpy(), clean.cpu().numpy()) <= ATTN_RTOL


@pytest.mark.parametrize("H,HKV,n_seq,most", [(8, 8, 1500, 80), (2, 1, 1200, 30), (40, 8, 700, 40)])
def test_many_sequences(gpu, H, HKV, n_seq, most):
    """More sequences than the plan holds in shared memory, more units on a line than it does, and too many
    of both to be sorted."""
    rng = np.random.default_rng(n_seq)
    lens = [int(x) for x in rng.integers(0, most + 1, n_seq)]
    _, q, k, v = _prompts(H, HKV, lens, 104)
    out = _run_prompts(gpu, q, k, v, lens, H, HKV)
    # one causal block-diagonal softmax per head in 64 bits, a few hundred rows at a time
    cu = _cu(lens)
    pick = sorted(set(rng.integers(0, n_seq, 60).tolist()) | {0, n_seq - 1})
    for s in pick:
        if lens[s]:
            r = slice(int(cu[s]), int(cu[s + 1]))
            _check_prompts(out[r], q[r], k[r], v[r], [lens[s]], H, HKV)
    assert torch.isfinite(out).all()


def test_other_batches_on_one_plan_buffer(gpu):
    """A buffer made for a large batch serves smaller ones after it, and the large one again."""
    H, HKV = 16, 8
    b = gpu.PackedBatch(20, 900, H, HKV)
    for lens in ([400, 500], [1] * 20, [33], [0, 0, 12], [400, 500]):
        _, q, k, v = _prompts(H, HKV, lens, 105)
        b.plan(_i32(_cu(lens)), sum(lens), max(lens))
        _check_prompts(gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV)), q, k, v, lens, H, HKV)


def test_one_plan_on_two_streams(gpu):
    """A plan is only read by the calls: two workspaces, two streams, one plan."""
    from exactinfer_amd import _capi
    H, HKV, lens = 16, 8, [300, 20, 1, 700]
    rows = sum(lens)
    _, q, k, v = _prompts(H, HKV, lens, 106)
    b = gpu.PackedBatch(4, rows, H, HKV)
    b.plan(_i32(_cu(lens)), rows, 700)
    ref = gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV))
    torch.cuda.synchronize()
    streams, outs, spaces = [torch.cuda.Stream() for _ in range(2)], [], []
    for s in streams:
        outs.append(torch.zeros_like(ref))
        spaces.append(torch.empty_like(b.ws))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, w in zip(streams, outs, spaces):
            _capi.call("ei_attn_packed", s.cuda_stream, q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(),
                       k.stride(0), o.data_ptr(), 4, rows, H, HKV, D, float(gpu.default_scale()), b.buf.data_ptr(),
                       b.nbytes, w.data_ptr(), b.ws_nbytes)
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def _pool(lens, kv, HKV, bs, seed, shared=0, spare=3, slack=1):
    """A pool of shuffled blocks, block table and every sequence's pool rows."""
    rng = np.random.default_rng(seed)
    need = [(t + bs - 1) // bs for t in kv]
    common = shared // bs
    total = common + sum(max(n - common, 0) for n in need) + spare
    order = rng.permutation(total)
    table = np.full((len(lens), max(need + [1]) + slack), -1, np.int32)
    at, rows = common, []
    for s, n in enumerate(need):
        own = max(n - common, 0)
        blocks = np.concatenate([order[:min(n, common)], order[at:at + own]])
        at += own
        table[s, :n] = blocks
        t = np.arange(kv[s])
        rows.append(torch.from_numpy((blocks[t // bs] * bs + t % bs).astype(np.int64)).cuda() if kv[s] else None)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn((total * bs, HKV, D), generator=g, device="cuda")
    v = torch.randn((total * bs, HKV, D), generator=g, device="cuda")
    return k, v, torch.from_numpy(table).cuda(), rows


CHUNKS = [  # H, HKV, block, lens, kv_len
    (8, 8, 32, [1], [1]), (16, 8, 64, [1] * 7, [1, 31, 32, 33, 64, 65, 700]),
    (16, 8, 64, [1, 100, 1, 60, 1], [301, 612, 34, 60, 901]), (40, 8, 32, [5] * 6, [29, 64, 101, 256, 300, 5]),
    (32, 8, 128, [130, 40], [1300, 40]), (8, 1, 256, [17, 0, 3], [500, 77, 1000]), (64, 8, 32, [3, 33], [400, 33]),
    (16, 8, 32, [6, 9, 3, 1], [2, 0, 3, 0]), (18, 6, 64, [2, 70], [4000, 333]), (8, 2, 64, [1, 1], [9000, 12]),
]


@pytest.mark.parametrize("H,HKV,bs,lens,kv", CHUNKS)
def test_paged_chunks(gpu, H, HKV, bs, lens, kv):
    kc, vc, table, rows_of = _pool(lens, kv, HKV, bs, 21)
    # what the pool holds beyond a sequence's keys must not matter
    own = torch.zeros(kc.shape[0], dtype=torch.bool, device="cuda")
    for r in rows_of:
        if r is not None:
            own[r] = True
    kc[~own], vc[~own] = float("nan"), float("inf")
    rows = sum(lens)
    q = torch.randn((rows, H * D), generator=torch.Generator(device="cuda").manual_seed(22), device="cuda")
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(_cu(lens)), rows, max(kv), kv_len=_i32(kv))
    out = gpu.attn_packed_paged(q, kc, vc, table, bs, b, gpu.AttnShape(H, HKV))
    cu = _cu(lens)
    for s, n in enumerate(lens):
        if n == 0:
            continue
        got = out[int(cu[s]):int(cu[s + 1])].cpu().numpy()
        if kv[s] == 0:
            assert np.all(got == 0.0)
            continue
        ref = _attend64(q[int(cu[s]):int(cu[s + 1])].double().view(n, H, D), kc[rows_of[s]].double(),
                        vc[rows_of[s]].double(), kv[s]).cpu().numpy()
        blind = max(0, n - kv[s])
        assert np.all(got[:blind] == 0.0)
        assert rel_err(got, ref) <= ATTN_RTOL, s


@pytest.mark.parametrize("H,HKV,lens", [(8, 2, [4, 5, 6, 8, 1]), (5, 1, [3, 4, 5, 6]), (8, 1, [2, 3, 4]),
                                        (4, 2, [8, 9, 10, 11]), (8, 2, [1, 1, 1]), (2, 1, [2, 1, 2]),
                                        (1, 1, [4, 5, 3])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_values_beside_few_rows(gpu, H, HKV, lens, bad):
    """1 to 32 rows of a KV head, with a bad key row or value that only the last two rows of each sequence
    see: the others keep their outputs, and a value's column alone is bad."""
    kv = [300 + 13 * i for i in range(len(lens))]
    kc, vc, table, rows_of = _pool(lens, kv, HKV, 32, 23)
    rows, cu = sum(lens), _cu(lens)
    q = torch.randn((rows, H * D), generator=torch.Generator(device="cuda").manual_seed(24), device="cuda")
    shape = gpu.AttnShape(H, HKV)
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(cu), rows, max(kv), kv_len=_i32(kv))
    clean = gpu.attn_packed_paged(q, kc, vc, table, 32, b, shape)
    for s, n in enumerate(lens):
        r = slice(int(cu[s]), int(cu[s + 1]))
        ref = _attend64(q[r].double().view(n, H, D), kc[rows_of[s]].double(), vc[rows_of[s]].double(), kv[s])
        assert rel_err(clean[r].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s
    at = torch.stack([rows_of[s][kv[s] - 2] for s in range(len(lens))])
    sees = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        sees[max(int(cu[s]), int(cu[s + 1]) - 2):int(cu[s + 1])] = True
    k2, v2 = kc.clone(), vc.clone()
    k2[at] = float("nan")
    out = gpu.attn_packed_paged(q, k2, vc, table, 32, b, shape)
    assert torch.isnan(out[sees]).all()
    if not sees.all():
        assert rel_err(out[~sees].cpu().numpy(), clean[~sees].cpu().numpy()) <= ATTN_RTOL
    v2[at, 0, 37] = bad
    out = gpu.attn_packed_paged(q, kc, v2, table, 32, b, shape)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[:, :H // HKV, 37] = sees[:, None]
    assert torch.equal(~torch.isfinite(out), hit)
    assert rel_err(torch.where(hit, clean, out).cpu().numpy(), clean.cpu().numpy()) <= ATTN_RTOL


def test_missing_pages_count_as_zeros(gpu):
    """Entries outside the pool and keys past the table: zeros, and nothing is read there."""
    H, HKV, bs = 16, 8, 32
    lens, kv = [3, 2, 1], [160, 100, 300]
    kc, vc, table, rows_of = _pool([3, 2, 1], [160, 100, 100], HKV, bs, 31, slack=0)  # 5 blocks: 160 keys at most
    table[0, 1], table[1, 3], table[0, 4] = -1, 10 ** 9, -2 ** 31
    q = torch.randn((6, H * D), generator=torch.Generator(device="cuda").manual_seed(32), device="cuda")
    b = gpu.PackedBatch(3, 6, H, HKV)
    b.plan(_i32(_cu(lens)), 6, 300, kv_len=_i32(kv))
    out = gpu.attn_packed_paged(q, kc, vc, table, bs, b, gpu.AttnShape(H, HKV))
    tab, cu = table.cpu().numpy(), _cu(lens)
    for s, n in enumerate(lens):
        k64 = torch.zeros((kv[s], HKV, D), dtype=torch.float64, device="cuda")
        v64 = torch.zeros_like(k64)
        for t in range(kv[s]):
            blk = int(tab[s, t // bs]) if t // bs < tab.shape[1] else -1
            if 0 <= blk < kc.shape[0] // bs:
                k64[t], v64[t] = kc[blk * bs + t % bs].double(), vc[blk * bs + t % bs].double()
        ref = _attend64(q[int(cu[s]):int(cu[s + 1])].double().view(n, H, D), k64, v64, kv[s])
        assert rel_err(out[int(cu[s]):int(cu[s + 1])].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s


def _norm_rope64(x, gamma, pos, rd, theta=1e6, eps=1e-6):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    f = theta ** (-2.0 * torch.arange(rd // 2, device=x.device, dtype=torch.float64) / rd)
    th = pos.double()[:, None, None] * f
    a, b = y[..., :rd // 2], y[..., rd // 2:rd]
    return torch.cat([a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos(), y[..., rd:]], -1)


@pytest.mark.parametrize("H,HKV,bs,lens,kv,rd", [
    (16, 8, 64, [1, 100, 1, 60, 1], [301, 612, 34, 60, 901], 128),
    (32, 8, 32, [5] * 6, [29, 64, 101, 256, 300, 5], 128), (40, 8, 128, [130, 1], [131, 1], 64),
    (8, 1, 32, [0, 7, 33], [40, 39, 33], 126), (64, 8, 64, [3, 3], [3, 400], 128),
])
def test_step(gpu, H, HKV, bs, lens, kv, rd):
    kc, vc, table, rows_of = _pool(lens, kv, HKV, bs, 41)
    shape = gpu.AttnShape(H, HKV, rope_dim=rd)
    rows, cu = sum(lens), _cu(lens)
    g = torch.Generator(device="cuda").manual_seed(42)
    qkv = torch.randn((rows, shape.qkv + 64), generator=g, device="cuda")
    qg, kg = 1 + 0.1 * torch.randn(D, generator=g, device="cuda"), 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    cs = gpu.rope_table_scaled(max(kv), rd)
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(cu), rows, max(kv), kv_len=_i32(kv))
    k0, v0, raw = kc.clone(), vc.clone(), qkv.clone()
    out = gpu.packed_step_paged(qkv, kc, vc, table, bs, b, shape, qg, kg, cs)
    assert torch.equal(qkv, raw)
    written = torch.zeros(kc.shape[0], dtype=torch.bool, device="cuda")
    x = raw[:, :shape.qkv].double().view(rows, H + 2 * HKV, D)
    k64, v64 = k0.double(), v0.double()
    for s, n in enumerate(lens):
        if n == 0:
            continue
        r = slice(int(cu[s]), int(cu[s + 1]))
        pos = torch.arange(kv[s] - n, kv[s], device="cuda")
        new = rows_of[s][kv[s] - n:]
        written[new] = True
        k64[new] = _norm_rope64(x[r, H:H + HKV], kg, pos, rd)
        v64[new] = x[r, H + HKV:]
        # an element within 8.2 half steps of its pair's length, a pair at most sqrt(2 * 128) gammas long
        assert (kc[new].double() - k64[new]).abs().max() <= 8.2 * 2 ** -24 * 16 * kg.abs().max()
        assert torch.equal(vc[new].double(), v64[new])
        q64 = _norm_rope64(x[r, :H], qg, pos, rd)
        ref = _attend64(q64, k64[rows_of[s]], v64[rows_of[s]], kv[s])
        assert rel_err(out[r].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s
    assert torch.equal(kc[~written], k0[~written]) and torch.equal(vc[~written], v0[~written])


def test_step_outside_table_and_pages(gpu):
    """Rows at positions outside the table, or whose page is missing, append nothing."""
    H, HKV, bs = 16, 8, 32
    lens, kv = [4, 3, 3], [3, 70, 62]  # the first row of sequence 0 is at -1; sequence 1 passes the table
    kc, vc, table, _ = _pool(lens, kv, HKV, bs, 51, slack=0)
    table[2, 1] = -1  # positions 32 .. 63 of sequence 2
    shape = gpu.AttnShape(H, HKV)
    g = torch.Generator(device="cuda").manual_seed(52)
    qkv = torch.randn((10, shape.qkv), generator=g, device="cuda")
    one = torch.ones(D, device="cuda")
    cs = gpu.rope_table_scaled(68)  # positions 68, 69 are past it
    b = gpu.PackedBatch(3, 10, H, HKV)
    b.plan(_i32(_cu(lens)), 10, 100, kv_len=_i32(kv))
    k0 = kc.clone()
    out = gpu.packed_step_paged(qkv, kc, vc, table, bs, b, shape, one, one, cs)
    tab = table.cpu().numpy()
    changed = (kc != k0).flatten(1).any(1).nonzero().flatten().tolist()
    want = sorted([int(tab[0, 0]) * bs + p for p in (0, 1, 2)] + [int(tab[1, 67 // bs]) * bs + 67 % bs])
    assert changed == want
    assert (out[0] == 0).all() and torch.isfinite(out).all()


def test_prompts_chunks_and_decode_together(gpu):
    """A run as a serving program makes it: two prompts packed and attended over their own rows and put
    into the pool by the step, then chunks and single tokens through it, against the sequences one at a time."""
    H, HKV, bs = 32, 8, 64
    shape = gpu.AttnShape(H, HKV)
    lens0, more = [150, 70], [[1, 40], [1, 1], [3, 1]]
    total = [sum([lens0[s]] + [m[s] for m in more]) for s in range(2)]
    kc, vc, table, rows_of = _pool(lens0, total, HKV, bs, 61)
    g = torch.Generator(device="cuda").manual_seed(62)
    seqs = [torch.randn((t, shape.qkv), generator=g, device="cuda") for t in total]
    qg, kg = 1 + 0.1 * torch.randn(D, generator=g, device="cuda"), 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    cs = gpu.rope_table_scaled(max(total))
    b = gpu.PackedBatch(2, sum(lens0), H, HKV)
    outs, at = [[], []], [0, 0]
    for step, lens in enumerate([lens0] + more):
        rows = torch.cat([seqs[s][at[s]:at[s] + lens[s]] for s in range(2)])
        at = [at[s] + lens[s] for s in range(2)]
        b.plan(_i32(_cu(lens)), sum(lens), max(total), kv_len=_i32(at))
        out = gpu.packed_step_paged(rows, kc, vc, table, bs, b, shape, qg, kg, cs)
        if step == 0:
            # the same prompts without a cache: norm and turn, then attention over the rows themselves
            pos = _i32(np.concatenate([np.arange(n) for n in lens]))
            qk = rows.clone()
            gpu.rope_rows(qk, H, cs, pos, gamma=qg, out=qk)
            keys = qk[:, H * D:]
            gpu.rope_rows(keys, HKV, cs, pos, gamma=kg, out=keys)
            b.plan(_i32(_cu(lens)), sum(lens), max(lens))
            alone = gpu.attn_packed(qk, keys, qk[:, (H + HKV) * D:], b, shape)
            assert rel_err(alone.cpu().numpy(), out.cpu().numpy()) <= ATTN_RTOL
        for s, o in enumerate(out.split(lens)):
            outs[s].append(o)
    for s in range(2):
        x = seqs[s].double().view(total[s], H + 2 * HKV, D)
        pos = torch.arange(total[s], device="cuda")
        q, k = _norm_rope64(x[:, :H], qg, pos, D), _norm_rope64(x[:, H:H + HKV], kg, pos, D)
        ref = _attend64(q, k, x[:, H + HKV:], total[s])
        assert rel_err(torch.cat(outs[s]).cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL
    # and one more token of both through the decode step on the same pool
    ws = gpu.DecodeWorkspace(2, H, HKV, max(total))
    row = torch.stack([seqs[s][-1] for s in range(2)])
    dec = gpu.decode_step_paged(row, kc, vc, table, bs, _i32(total), shape, qg, kg, cs, ws)
    assert rel_err(dec.cpu().numpy(), torch.stack([outs[s][-1][-1] for s in range(2)]).cpu().numpy()) <= ATTN_RTOL


def test_captured_step_replays_with_new_lengths(gpu):
    """The plan and the step in one graph: lengths, tables and rows change between replays."""
    H, HKV, bs, n_seq = 16, 8, 64, 3
    shape = gpu.AttnShape(H, HKV)
    lens = [[1, 60, 1], [20, 1, 1], [1, 1, 0]]
    kv = [[200, 60, 33], [300, 61, 34], [301, 62, 0]]
    kc, vc, table, rows_of = _pool(lens[0], [320, 70, 40], HKV, bs, 71)
    rows = 64
    g = torch.Generator(device="cuda").manual_seed(72)
    one = torch.ones(D, device="cuda")
    cs = gpu.rope_table_scaled(400)
    b = gpu.PackedBatch(n_seq, rows, H, HKV)
    qkv = torch.randn((rows, shape.qkv), generator=g, device="cuda")
    cu, kl = _i32(_cu(lens[0])), _i32(kv[0])
    out = torch.zeros((rows, H, D), device="cuda")

    def step():
        b.plan(cu, rows, 400, kv_len=kl)
        gpu.packed_step_paged(qkv, kc, vc, table, bs, b, shape, one, one, cs, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rnd in range(6):
        i = rnd % 3
        cu.copy_(_i32(_cu(lens[i])))
        kl.copy_(_i32(kv[i]))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        k0, v0 = kc.clone(), vc.clone()
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        replayed, k1, v1 = out.clone(), kc.clone(), vc.clone()
        kc.copy_(k0), vc.copy_(v0)
        out.fill_(9.0)
        step()
        torch.cuda.synchronize()
        assert torch.equal(replayed, out) and torch.equal(k1, kc) and torch.equal(v1, vc)
        n = sum(lens[i])
        assert (out[n:] == 9.0).all() and torch.isfinite(out[:n]).all()


def test_another_stream(gpu):
    H, HKV, lens = 16, 8, [90, 200]
    _, q, k, v = _prompts(H, HKV, lens, 81)
    shape = gpu.AttnShape(H, HKV)
    b = gpu.PackedBatch(2, 290, H, HKV)
    b.plan(_i32(_cu(lens)), 290, 200)
    ref = gpu.attn_packed(q, k, v, b, shape)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b2 = gpu.PackedBatch(2, 290, H, HKV)
        b2.plan(_i32(_cu(lens)), 290, 200)
        got = gpu.attn_packed(q, k, v, b2, shape)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref)


def test_python_refusals(gpu):
    H, HKV = 16, 8
    shape = gpu.AttnShape(H, HKV)
    _, q, k, v = _prompts(H, HKV, [8], 91)
    b = gpu.PackedBatch(2, 8, H, HKV)
    with pytest.raises(ValueError, match="no plan"):
        gpu.attn_packed(q, k, v, b, shape)
    for match, args, kw in (("int32", (_i32([0, 8]).long(), 8, 8), {}), ("made for", (_i32([0, 8]), 9, 8), {}),
                            ("made for", (_i32([0, 1, 2, 8]), 8, 8), {}), ("made for", (_i32([0]), 8, 8), {}),
                            ("lengths", (_i32([0, 8]), 8, 8), dict(kv_len=_i32([8, 8]))),
                            ("GPU tensor", (torch.zeros(2, dtype=torch.int32), 8, 8), {})):
        with pytest.raises(ValueError, match=match):
            b.plan(*args, **kw)
    b.plan(_i32([0, 8]), 8, 8)
    with pytest.raises(ValueError, match="rows of"):
        gpu.attn_packed(q[:7], k, v, b, shape)
    with pytest.raises(ValueError, match="row stride"):
        gpu.attn_packed(q, k, v.contiguous(), b, shape)
    with pytest.raises(ValueError, match="heads"):
        gpu.attn_packed(q, k, v, b, gpu.AttnShape(32, 8))
    with pytest.raises(ValueError, match="float32"):
        gpu.attn_packed(q.double(), k, v, b, shape)
    pool = torch.zeros((64, HKV, D), device="cuda")
    with pytest.raises(ValueError, match="block_table"):
        gpu.attn_packed_paged(q, pool, pool, _i32([0, 1]), 32, b, shape)
    with pytest.raises(ValueError, match="pools of rows"):
        gpu.attn_packed_paged(q, pool, pool[:32], _i32([[0, 1]]), 32, b, shape)
    with pytest.raises(RuntimeError, match="block_size 16"):
        gpu.attn_packed_paged(q, pool, pool, _i32([[0, 1]]), 16, b, shape)
    b.plan(_i32([0, 8]), 8, 64, kv_len=_i32([20]))
    with pytest.raises(ValueError, match="whole prompts"):
        gpu.attn_packed(q, k, v, b, shape)
    b.plan(_i32([0, 0]), 0, 8)
    assert gpu.attn_packed(q, k, v, b, shape).shape == (0, H, D)
    with pytest.raises(ValueError, match="GPU tensor"):
        gpu.PackedBatch(2, 8, H, HKV, device="cpu").plan(_i32([0, 8]), 8, 8)


def test_single_rows_of_any_stride(gpu):
    """The stride of a one-row view is not used: rows of buffers whose width is no multiple of four serve, and
    keys and values of buffers of different widths."""
    H, HKV = 16, 8
    _, q, k, v = _prompts(H, HKV, [1], 92)
    q1, k1 = torch.zeros((3, H * D + 1), device="cuda")[:1, :H * D], torch.zeros((2, HKV * D + 64), device="cuda")[:1]
    q1.copy_(q)
    k1[:, :HKV * D].copy_(k)
    b = gpu.PackedBatch(1, 1, H, HKV)
    b.plan(_i32([0, 1]), 1, 1)
    out = gpu.attn_packed(q1, k1[:, :HKV * D], v.contiguous(), b, gpu.AttnShape(H, HKV))
    assert torch.equal(out, gpu.attn_packed(q, k, v, b, gpu.AttnShape(H, HKV)))
    cs = gpu.rope_table_scaled(16, D, 1e6)
    pos = _i32([9])
    assert torch.equal(gpu.rope_rows(q1, H, cs, pos), gpu.rope_rows(q, H, cs, pos))


@pytest.mark.parametrize("H,HKV", [(7, 1), (18, 3), (30, 5), (14, 7), (300, 300), (264, 33), (6, 6)])
def test_any_number_of_heads(gpu, H, HKV):
    """KV heads that do not divide the GPU's units, more of them than it has, and every group's size."""
    lens = [3, 45, 1, 20] if H < 100 else [3, 33, 1]
    _, q, k, v = _prompts(H, HKV, lens, 111)
    _check_prompts(_run_prompts(gpu, q, k, v, lens, H, HKV), q, k, v, lens, H, HKV)
    kv = [n + 90 for n in lens]
    kc, vc, table, rows_of = _pool(lens, kv, HKV, 32, 112)
    b = gpu.PackedBatch(len(lens), sum(lens), H, HKV)
    b.plan(_i32(_cu(lens)), sum(lens), max(kv), kv_len=_i32(kv))
    out = gpu.attn_packed_paged(q, kc, vc, table, 32, b, gpu.AttnShape(H, HKV))
    for s, (a, n) in enumerate(zip(_cu(lens), lens)):
        r = slice(int(a), int(a) + n)
        ref = _attend64(q[r].double().view(n, H, D), kc[rows_of[s]].double(), vc[rows_of[s]].double(), kv[s])
        assert rel_err(out[r].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s


def test_batches_without_rows_or_keys(gpu):
    """Rows that belong to nobody stay; rows of sequences without keys are zeros, lengths below 0 count as 0 and
    lengths above max_kv as max_kv."""
    H, HKV = 16, 8
    shape = gpu.AttnShape(H, HKV)
    _, q, k, v = _prompts(H, HKV, [6], 113)
    b = gpu.PackedBatch(3, 6, H, HKV)
    mark = torch.full((6, H, D), 7.5, device="cuda")
    b.plan(_i32([0, 0, 0, 0]), 6, 10)
    out = gpu.attn_packed(q, k, v, b, shape, out=mark.clone())
    assert torch.equal(out, mark)
    b.plan(_i32([0, 2, 2, 5]), 6, 0)
    out = gpu.attn_packed(q, k, v, b, shape, out=mark.clone())
    assert (out[:5] == 0).all() and torch.equal(out[5:], mark[5:])
    kc, vc, table, rows_of = _pool([2, 1, 3], [40, 1, 50], HKV, 32, 114)
    b.plan(_i32([0, 2, 3, 6]), 6, 50, kv_len=_i32([40, -5, 2 ** 31 - 1]))
    out = gpu.attn_packed_paged(q, kc, vc, table, 32, b, shape)
    assert (out[2] == 0).all()
    b.plan(_i32([0, 2, 3, 6]), 6, 50, kv_len=_i32([40, 0, 50]))
    assert torch.equal(out, gpu.attn_packed_paged(q, kc, vc, table, 32, b, shape))
    qg = torch.ones(D, device="cuda")
    qkv = torch.randn((6, shape.qkv), device="cuda")
    cs = gpu.rope_table_scaled(64)
    b.plan(_i32([0, 0, 0, 0]), 6, 50, kv_len=_i32([40, 1, 50]))
    k0, v0 = kc.clone(), vc.clone()
    out = gpu.packed_step_paged(qkv, kc, vc, table, 32, b, shape, qg, qg, cs, out=mark.clone())
    assert torch.equal(out, mark) and torch.equal(kc, k0) and torch.equal(vc, v0)


def test_blocks_past_32_bits(gpu):
    """Pool rows beyond 2^31 values and 2^32 bytes, appended and read."""
    H, HKV, bs = 16, 8, 256
    n_blocks = 2 ** 31 // (HKV * D * bs) + 6
    kc = torch.empty((n_blocks * bs, HKV, D), device="cuda")
    vc = torch.empty_like(kc)
    lens, kv = [1, 40], [300, 200]
    table = _i32([[n_blocks - 1, n_blocks - 4], [n_blocks // 2 + 3, 0]])
    rows_of = [torch.cat([torch.arange(bs) + int(e) * bs for e in row])[:kv[s]].cuda()
               for s, row in enumerate(table.tolist())]
    g = torch.Generator(device="cuda").manual_seed(115)
    for r in rows_of:
        kc[r] = torch.randn((len(r), HKV, D), generator=g, device="cuda")
        vc[r] = torch.randn((len(r), HKV, D), generator=g, device="cuda")
    shape = gpu.AttnShape(H, HKV)
    qkv = torch.randn((41, shape.qkv), generator=g, device="cuda")
    one = torch.ones(D, device="cuda")
    b = gpu.PackedBatch(2, 41, H, HKV)
    b.plan(_i32(_cu(lens)), 41, 300, kv_len=_i32(kv))
    out = gpu.packed_step_paged(qkv, kc, vc, table, bs, b, shape, one, one, gpu.rope_table_scaled(512))
    x = qkv.double().view(41, H + 2 * HKV, D)
    for s, (a, n) in enumerate(zip(_cu(lens), lens)):
        r = slice(int(a), int(a) + n)
        new = rows_of[s][kv[s] - n:]
        assert torch.equal(vc[new], qkv[r].view(n, -1, D)[:, H + HKV:])
        pos = torch.arange(kv[s] - n, kv[s], device="cuda")
        q64 = _norm_rope64(x[r, :H], one, pos, D)
        ref = _attend64(q64, kc[rows_of[s]].double(), vc[rows_of[s]].double(), kv[s])
        assert rel_err(out[r].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s


def test_keys_and_values_in_one_pool(gpu):
    """A pool may serve as keys and values where it is only read, and sequences may list the same block twice."""
    H, HKV, bs = 16, 8, 32
    lens, kv = [5, 1], [90, 70]
    kc, _, table, _ = _pool(lens, kv, HKV, bs, 116)
    table[0, 1] = table[0, 0]
    table[1] = table[0]
    b = gpu.PackedBatch(2, 6, H, HKV)
    b.plan(_i32(_cu(lens)), 6, 90, kv_len=_i32(kv))
    q = torch.randn((6, H * D), generator=torch.Generator(device="cuda").manual_seed(117), device="cuda")
    out = gpu.attn_packed_paged(q, kc, kc, table, bs, b, gpu.AttnShape(H, HKV))
    for s, (a, n) in enumerate(zip(_cu(lens), lens)):
        t = np.arange(kv[s])
        rows = torch.from_numpy(table[s].cpu().numpy().astype(np.int64)[t // bs] * bs + t % bs).cuda()
        x = kc[rows].double()
        ref = _attend64(q[int(a):int(a) + n].double().view(n, H, D), x, x, kv[s])
        assert rel_err(out[int(a):int(a) + n].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s
