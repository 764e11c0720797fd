"""GPU tests of the rule by which the plan of a packed batch shares out its work (include/ei_packed.h), made again
from the lengths."""
import numpy as np
import pytest

from tests.test_gpu_packed import BATCHES, _cu, _i32, _read_plan, _shares

pytestmark = pytest.mark.gpu

ONCE = 5              # tiles that a unit's pass costs besides its own
SLACK = 32            # whole units may pass an equal share by 1/32
TURNS = {False: 2, True: 8}

MORE = [  # H, HKV, lens, kv_len (None: whole prompts): all rounds dealt, all but one, none; even and uneven ones
    (32, 8, [250] * 8, None), (32, 8, [2048], None), (40, 8, [900, 700], None), (32, 8, [1500], [9500]),
    (32, 8, [1024, 400], [31024, 400]), (32, 8, [64] + [32] * 64, [30064] + [32] * 64),
    (16, 8, [256] + [200] * 30, [30256] + [200] * 30), (64, 8, [600, 300, 200], [9600, 300, 200]),
    (8, 8, [130] * 200, [300 + 7 * i for i in range(200)]), (16, 2, [777] * 5, None),
]


@pytest.mark.parametrize("H,HKV,lens,kv", BATCHES + MORE)
def test_rounds_and_shares(gpu, H, HKV, lens, kv):
    """Whole units are dealt in descending order as long as full rounds of them last; the last full round only if no
    workgroup then has more than an equal share of everything and 1/32; and beyond what was dealt to it no
    workgroup gets more of the lines than what is missing to an equal share.

    A cut is moved by less than a turn of tiles and then at most to `keep` = 5 or 8 tiles beyond (or to an end of a
    unit shorter than twice that), its pass included, and a cut unit's second part costs a pass of its own: a share
    has at most two moved cuts and one such part."""
    rows, N, G = sum(lens), _shares(HKV), H // HKV
    b = gpu.PackedBatch(len(lens), rows, H, HKV)
    b.plan(_i32(_cu(lens)), rows, max(kv or lens), kv_len=None if kv is None else _i32(kv))
    head, wide, wide_shares, few, few_shares = _read_plan(b, lens, rows, H, HKV)
    cost = {False: wide[:, 5].astype(int) + ONCE, True: few[:, 5].astype(int) + ONCE}
    both = -(-(int(cost[False].sum()) + int(cost[True].sum())) // N)
    full = len(wide) // N if len(wide) * len(lens) <= 1 << 20 else 0

    def dealt(rounds):
        load = np.zeros(N, int)
        for r in range(rounds):
            load[::-1 if r % 2 else 1] += cost[False][r * N:(r + 1) * N]
        return load

    rounds = full - (full > 0 and dealt(full).max() > both + both // SLACK)
    assert head[6] == rounds and head[7] == rounds * N and head[8] == len(wide) - rounds * N and head[9] == len(few)
    if rounds and rounds == full:
        assert dealt(rounds).max() <= both + both // SLACK
    load = dealt(rounds)
    for is_few, units, shares, first in ((False, wide, wide_shares, rounds * N), (True, few, few_shares, 0)):
        want = np.maximum(load, both if is_few else -(-int(cost[False].sum()) // N))
        n, tiles = len(units) - first, units[first:, 5].astype(int)
        for j, (a, ta, e, te) in enumerate(shares[:, :4].tolist()):
            for i in range(a, min(e + 1, n)):
                lo, hi = (ta if i == a else 0), (te if i == e else tiles[i])
                if i < e or te > 0:
                    load[j] += hi - lo + ONCE
        assert np.all(load <= want + 2 * (TURNS[is_few] + max(TURNS[is_few], ONCE) + ONCE) + ONCE), is_few
