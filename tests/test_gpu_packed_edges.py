"""GPU tests of the packed batch (include/ei_packed.h) at the edges of its arithmetic and of its lengths, against
softmax attention in 64 bits; the bar is that of tests/test_gpu_packed.py unless a test derives its own."""
import numpy as np
import pytest
import torch

from tests.parity import ATTN_RTOL, rel_err
from tests.test_gpu_packed import (D, SCALE, _attend64, _check_prompts, _cu, _i32, _norm_rope64, _pool, _prompts,
                                   _read_plan, _run_prompts)

pytestmark = pytest.mark.gpu


def _paged(gpu, q, kc, vc, table, bs, lens, kv, H, HKV, scale=None):
    b = gpu.PackedBatch(len(lens), sum(lens), H, HKV)
    b.plan(_i32(_cu(lens)), sum(lens), max(kv), kv_len=_i32(kv))
    return b, gpu.attn_packed_paged(q, kc, vc, table, bs, b, gpu.AttnShape(H, HKV), scale=scale)


def _check_paged(out, q, kc, vc, rows_of, lens, kv, H, scale=SCALE, tol=ATTN_RTOL):
    for s, (a, n) in enumerate(zip(_cu(lens), lens)):
        r = slice(int(a), int(a) + n)
        ref = _attend64(q[r].double().view(n, H, D), kc[rows_of[s]].double(), vc[rows_of[s]].double(), kv[s], scale)
        e = rel_err(out[r].cpu().numpy(), ref.cpu().numpy())
        assert e <= tol, (s, e)


@pytest.mark.parametrize("H,HKV,n", [(8, 1, 16), (32, 8, 64), (8, 1, 1), (16, 8, 1), (32, 8, 5)])
@pytest.mark.parametrize("T", [3000, 5000, 9000])
def test_infinite_value_in_the_last_part(gpu, H, HKV, n, T):
    """Wide and few-row units cut into parts whose number is whatever it is: an infinity that every row sees in the
    last part reaches the output as it is."""
    kc, vc, table, rows_of = _pool([n], [T], HKV, 64, 201)
    q = torch.randn((n, H * D), generator=torch.Generator(device="cuda").manual_seed(202), device="cuda")
    at = rows_of[0][T - n]
    vc[at, 0, 5], vc[at, 0, 70] = float("inf"), float("-inf")
    b, out = _paged(gpu, q, kc, vc, table, 64, [n], [T], H, HKV)
    _, _, wide, _, few = _read_plan(b, [n], n, H, HKV)
    assert (wide[:, 4] > 0).any() or (few[:, 4] > 0).any()  # (a unit is cut)
    G = H // HKV
    assert (out[:, :G, 5] == float("inf")).all() and (out[:, :G, 70] == float("-inf")).all()
    vc[at, 0, 5] = vc[at, 0, 70] = 0.0
    ref = _attend64(q.double().view(n, H, D), kc[rows_of[0]].double(), vc[rows_of[0]].double(), T)
    out[:, :G, 5], out[:, :G, 70] = ref[:, :G, 5].float(), ref[:, :G, 70].float()
    assert rel_err(out.cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL


@pytest.mark.parametrize("H,HKV,lens", [(16, 8, [100, 7, 300]), (8, 1, [60]), (32, 8, [4, 8, 1])])
@pytest.mark.parametrize("e", [-104, -108, -112])
@pytest.mark.parametrize("signs", ["any", "against", "one key"])
def test_tiny_queries_of_huge_keys(gpu, H, HKV, lens, e, signs):
    """q of about 2^e against keys of about 2^-e: the scores are ordinary, whatever lies between, also where all of a
    row are negative, or a single key is huge."""
    _, q, k, v = _prompts(H, HKV, lens, 203)
    if signs != "any":
        q, k = -q.abs(), k.abs()
    if signs == "one key":
        k[1:], k[0] = 0.0, k[0] * 0.25
    q, k, v = (q * 2.0 ** e).contiguous(), (k * 2.0 ** -e).contiguous(), v.contiguous()
    _check_prompts(_run_prompts(gpu, q, k, v, lens, H, HKV), q, k, v, lens, H, HKV)


def _sink_batch(gpu, T, n_seq, seed):
    """n_seq sequences of 16 new rows over the same T keys, zero but for channel 0, with values about 1: one sequence of
    a single KV head, cut into parts, or 32 of eight heads, in whole units.

    In a whole unit each of two accumulators is rounded twice in each of six matrix instructions per 64 keys, by at
    most 2^-24 of the sum so far, half of the last one on the average.  Equal weights round alike: 12 T / 64 * 2^-25
    on top of the bar (whose signs are random)."""
    H, HKV, n = (8, 1, 16) if n_seq == 1 else (64, 8, 16)
    tol = ATTN_RTOL + (0 if n_seq == 1 else 12 * T / 64 * 2.0 ** -25)
    kc, vc, table, rows_of = _pool([n], [T], HKV, 64, seed)
    r = rows_of[0]
    kc[r] = 0.0
    vc[r] = vc[r] * 0.25 + 1.0
    q = torch.randn((n * n_seq, H * D), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
    q[:, ::D] = 8.0

    def run():
        b, out = _paged(gpu, q, kc, vc, table.repeat(n_seq, 1), 64, [n] * n_seq, [T] * n_seq, H, HKV, scale=0.125)
        head, _, wide, _, _ = _read_plan(b, [n] * n_seq, n * n_seq, H, HKV)
        assert head[6] == 1 if n_seq > 1 else T < 200 or (wide[:, 4] > 0).any()
        for s in (0, n_seq - 1):
            _check_paged(out[n * s:n * s + n], q[n * s:n * s + n], kc, vc, rows_of, [n], [T], H, 0.125, tol)

    return kc, vc, r, n, run


@pytest.mark.parametrize("T", [64, 200, 2000, 8000, 30000])
@pytest.mark.parametrize("nats", [8.0, 12.0, 15.0, 16.3, 17.0, 17.7, 18.0, 20.0])
@pytest.mark.parametrize("sinks", ["first", "every tile"])
@pytest.mark.parametrize("n_seq", [1, 32])
def test_dominant_keys_with_no_value(gpu, T, nats, sinks, n_seq):
    """Keys that take nearly all of the weight and have a value of zero: the output is what the many equal small
    weights of the others give, so an error that they share does not average out.

    The scores are 8 * nats / 8 at the sinks and 0 elsewhere, each off by some 4 * 2^-24 of itself at most, up to 29
    in log2 units: weights by 29 * 2^-22 * ln 2 = 4.8e-6, all by the same."""
    kc, vc, r, n, run = _sink_batch(gpu, T, n_seq, 204)
    at = r[:1] if sinks == "first" else r[torch.arange(0, T - n + 1, 32, device="cuda")]
    kc[at, :, 0] = nats
    vc[at] = 0.0
    run()


@pytest.mark.parametrize("H,HKV,n", [(8, 8, 1), (32, 8, 1), (32, 8, 5), (32, 8, 8)])
@pytest.mark.parametrize("T", [3000, 30000])
@pytest.mark.parametrize("nats", [8.0, 12.0, 15.0, 18.0])
def test_dominant_key_before_few_rows(gpu, H, HKV, n, T, nats):
    """The same for single tokens and drafts of 64 sequences over one sequence's keys.

    A wave's accumulators are rounded in each of eight matrix instructions per 256 keys, by at most 2^-24 of the sum so
    far, half of the last one on the average, and equal weights round alike: T / 32 * 2^-25 on top of the bar."""
    kc, vc, table, rows_of = _pool([n], [T], HKV, 64, 215)
    r = rows_of[0]
    kc[r] = 0.0
    vc[r] = vc[r] * 0.25 + 1.0
    kc[r[0], :, 0] = nats
    vc[r[0]] = 0.0
    q = torch.randn((n * 64, H * D), generator=torch.Generator(device="cuda").manual_seed(216), device="cuda")
    q[:, ::D] = 8.0
    _, out = _paged(gpu, q, kc, vc, table.repeat(64, 1), 64, [n] * 64, [T] * 64, H, HKV, scale=0.125)
    for s in (0, 31, 63):
        rows = slice(n * s, n * s + n)
        _check_paged(out[rows], q[rows], kc, vc, rows_of, [n], [T], H, 0.125, ATTN_RTOL + T / 32 * 2.0 ** -25)


@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("step", [1.0, 3.0])
@pytest.mark.parametrize("n_seq", [1, 32])
def test_scores_that_fall_or_rise_over_the_tiles(gpu, up, step, n_seq):
    """Scores that fall or rise by `step` a tile, most of the weight without a value: the sums follow in both
    directions.  (Scores of at most 24: as above.)"""
    T = int(24 / step) * 32
    kc, vc, r, n, run = _sink_batch(gpu, T, n_seq, 206)
    level = torch.arange(T, device="cuda") // 32
    level = level if up else T // 32 - 1 - level
    kc[r, :, 0] = level[:, None].float() * step
    vc[r[level >= T // 64]] = 0.0
    run()


@pytest.mark.parametrize("H,HKV,lens", [(8, 1, [200]), (16, 8, [90, 300])])
@pytest.mark.parametrize("e", [10, 22, 30, 60])
def test_channels_that_meet_zeros(gpu, H, HKV, lens, e):
    """A channel of q and one of K 2^e times the others, each against zeros: the scores are those of the others."""
    _, q, k, v = (t.contiguous() for t in _prompts(H, HKV, lens, 208))
    q[:, 3::D] *= 2.0 ** e
    k[:, 3::D] = 0.0
    k[:, 77::D] *= 2.0 ** e
    q[:, 77::D] = 0.0
    _check_prompts(_run_prompts(gpu, q, k, v, lens, H, HKV), q, k, v, lens, H, HKV)


PAGED_WIDE = [  # H, HKV, lens, kv_len, whole units, cut ones
    (8, 2, [40, 70, 33], [300, 70, 700], False, True), (8, 1, [20], [4000], False, True),
    (16, 8, [60] * 64, [200 + i % 20 for i in range(64)], True, False),
]


@pytest.mark.parametrize("H,HKV,lens,kv,whole,cut", PAGED_WIDE)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_values_beside_many_rows(gpu, H, HKV, lens, kv, whole, cut, bad):
    """More than 32 rows of a KV head over shuffled pages, with a bad key row or value that only the last two rows of
    each sequence see: the others keep their outputs, and a value's column alone is bad."""
    kc, vc, table, rows_of = _pool(lens, kv, HKV, 32, 209)
    rows, cu, G = sum(lens), _cu(lens), H // HKV
    q = torch.randn((rows, H * D), generator=torch.Generator(device="cuda").manual_seed(210), device="cuda")
    b, clean = _paged(gpu, q, kc, vc, table, 32, lens, kv, H, HKV)
    head, _, wide, _, _ = _read_plan(b, lens, rows, H, HKV)
    assert not whole or head[6] > 0
    assert not cut or (wide[:, 4] > 0).any()
    _check_paged(clean, q, kc, vc, rows_of, lens, kv, H)
    at = torch.stack([rows_of[s][kv[s] - 2] for s in range(len(lens))])
    sees = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for s in range(len(lens)):
        sees[int(cu[s + 1]) - 2:int(cu[s + 1])] = True
    k2, v2 = kc.clone(), vc.clone()
    k2[at] = float("nan")
    _, out = _paged(gpu, q, k2, vc, table, 32, lens, kv, H, HKV)
    assert torch.isnan(out[sees]).all()
    assert rel_err(out[~sees].cpu().numpy(), clean[~sees].cpu().numpy()) <= ATTN_RTOL
    v2[at, 0, 37] = bad
    _, out = _paged(gpu, q, kc, v2, table, 32, lens, kv, H, HKV)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[:, :G, 37] = sees[:, None]
    assert torch.equal(torch.isnan(out) if bad != bad else out == bad, hit)
    assert rel_err(torch.where(hit, clean, out).cpu().numpy(), clean.cpu().numpy()) <= ATTN_RTOL


@pytest.mark.parametrize("H,HKV,lens,kv,whole,cut", PAGED_WIDE)
def test_large_value_of_a_light_key_over_pages(gpu, H, HKV, lens, kv, whole, cut):
    """A value row 2^30 times the others at a key of weight e^-22.6: its part of the outputs and theirs.

    Scores of up to 33 + 6 in log2 units are rounded by up to 2^-19 in each of 127 additions, a weight by that times
    ln 2 of itself, an output by twice as much of the largest ordinary value, and of the light key's part.  (Planes of
    V scaled to the large row would be off by 2^-25 of 2^-13 of it, 2^-6.)"""
    kc, vc, table, rows_of = _pool(lens, kv, HKV, 32, 211)
    q = torch.randn((sum(lens), H * D), generator=torch.Generator(device="cuda").manual_seed(212), device="cuda")
    q[:, ::D] = 32.0
    kc[:, :, 0] = 8.0
    for s in range(len(lens)):
        kc[rows_of[s][7], :, 0] = 0.0
        vc[rows_of[s][7]] *= 2.0 ** 30
    _, out = _paged(gpu, q, kc, vc, table, 32, lens, kv, H, HKV)
    for s, (a, n) in enumerate(zip(_cu(lens), lens)):
        r = slice(int(a), int(a) + n)
        k64, v64 = kc[rows_of[s]].double(), vc[rows_of[s]].double()
        ref = _attend64(q[r].double().view(n, H, D), k64, v64, kv[s])
        v64[7] = 0.0
        most = v64.abs().max() + (ref - _attend64(q[r].double().view(n, H, D), k64, v64, kv[s])).abs().max()
        assert (out[r] - ref).abs().max() <= 2 * 127 * 2.0 ** -19 * np.log(2) * most, s


@pytest.mark.parametrize("H,HKV,lens", [(16, 8, [100, 7, 300]), (8, 1, [60, 700]), (32, 8, [4, 8, 1])])
@pytest.mark.parametrize("e", [104, 110, 118])
def test_values_near_the_end_of_fp32(gpu, H, HKV, lens, e):
    """Values of up to 2^(e + 2): so are the outputs, and the sums on the way to them at most some tens of times that."""
    _, q, k, v = (t.contiguous() for t in _prompts(H, HKV, lens, 217))
    v *= 2.0 ** e
    _check_prompts(_run_prompts(gpu, q, k, v, lens, H, HKV), q, k, v, lens, H, HKV)
    v[::5] *= 2.0 ** -60  # (rows that see such values alone have the fp32 products)
    _check_prompts(_run_prompts(gpu, q, k, v, lens, H, HKV), q, k, v, lens, H, HKV)


@pytest.mark.parametrize("H,HKV,bs,lens,kv,max_kv", [
    (16, 8, 32, [1, 3, 40, 2], [51, 52, 90, 40], 50), (8, 1, 64, [30], [140], 128),
    (32, 8, 32, [2, 2], [2 ** 31 - 1, 64], 64), (8, 8, 32, [1] * 1100, [33 + i % 40 for i in range(1100)], 64),
])
def test_step_past_max_kv_leaves_the_pool(gpu, H, HKV, bs, lens, kv, max_kv):
    """Sequences longer than the plan's max_kv: rows at positions from max_kv on append nothing, rows below it stand
    where kv_len puts them, other sequences are as ever."""
    real = [min(t, 200) for t in kv]  # (pages for all of a sequence's rows: nothing else keeps them from the pool)
    kc, vc, table, rows_of = _pool(lens, real, HKV, bs, 213)
    shape = gpu.AttnShape(H, HKV)
    rows, cu = sum(lens), _cu(lens)
    g = torch.Generator(device="cuda").manual_seed(214)
    qkv = torch.randn((rows, shape.qkv), generator=g, device="cuda")
    one = torch.ones(D, device="cuda")
    cs = gpu.rope_table_scaled(256)
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(cu), rows, max_kv, kv_len=_i32(kv))
    k0, v0 = kc.clone(), vc.clone()
    out = gpu.packed_step_paged(qkv, kc, vc, table, bs, b, shape, one, one, cs)
    x = qkv.double().view(rows, H + 2 * HKV, D)
    written = torch.zeros(kc.shape[0], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        pos = torch.arange(kv[s] - n, kv[s])
        keep = pos[pos < max_kv].cuda()
        if len(keep) == 0:
            continue
        new = rows_of[s][keep]
        written[new] = True
        r = slice(int(cu[s]), int(cu[s]) + len(keep))
        assert torch.equal(vc[new], qkv[r].view(len(keep), -1, D)[:, H + HKV:]), s
        want = _norm_rope64(x[r, H:H + HKV], one, keep, D)
        assert (kc[new].double() - want).abs().max() <= 8.2 * 2 ** -24 * 16, s
    assert torch.equal(kc[~written], k0[~written]) and torch.equal(vc[~written], v0[~written])
    for s, n in enumerate(lens):
        if kv[s] <= max_kv and s < 40:
            r = slice(int(cu[s]), int(cu[s + 1]))
            q64 = _norm_rope64(x[r, :H], one, torch.arange(kv[s] - n, kv[s], device="cuda"), D)
            ref = _attend64(q64, kc[rows_of[s]].double(), vc[rows_of[s]].double(), kv[s])
            assert rel_err(out[r].cpu().numpy(), ref.cpu().numpy()) <= ATTN_RTOL, s
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("max_kv", [-1, 2 ** 30 + 1, 2 ** 32 + 8, -2 ** 32 + 8])
def test_max_kv_out_of_range_is_refused(gpu, max_kv):
    """Also where its lowest 32 bits are a length."""
    b = gpu.PackedBatch(1, 8, 16, 8)
    with pytest.raises(ValueError, match="max_kv"):
        b.plan(_i32([0, 8]), 8, max_kv, kv_len=_i32([8]))
