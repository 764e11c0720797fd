"""Refusals of include/ei_packed.h's entry points: every check that comes before a launch (CPU only)."""
import ctypes

import pytest

P = ctypes.c_void_p(1 << 20)  # never dereferenced: validation fails first


def _at(n):
    return ctypes.c_void_p((1 << 20) + n)


FAR = [ctypes.c_void_p((i + 2) << 40) for i in range(8)]  # addresses far apart
BIG = 1 << 38


def _refused(match, name, *args):
    from exactinfer_amd import _capi
    with pytest.raises(_capi.EiError, match=match) as e:
        _capi.call(name, *args)
    return e.value.code


def _scaling(**kw):
    from exactinfer_amd import _capi
    d = dict(kind=0, factor=1.0, n_trained=4096, beta_fast=32.0, beta_slow=1.0, attn_factor=0.0)
    d.update(kw)
    return ctypes.byref(_capi.RopeScalingC(*(d[k] for k in ("kind", "factor", "n_trained", "beta_fast", "beta_slow",
                                                            "attn_factor"))))


@pytest.mark.parametrize("match,args", [
    ("cs missing", (None, 16, 128, 1e6, None)),
    ("aligned", (_at(4), 16, 128, 1e6, None)),
    ("n_pos 0", (P, 0, 128, 1e6, None)),
    ("rope_dim 130", (P, 16, 130, 1e6, None)),
    ("rope_dim 7", (P, 16, 7, 1e6, None)),
    ("rope_dim 0", (P, 16, 0, 1e6, None)),
    ("theta", (P, 16, 128, 0.0, None)),
    ("theta", (P, 16, 128, float("nan"), None)),
    ("theta", (P, 16, 128, float("inf"), None)),
])
def test_table_arguments(match, args):
    _refused(match, "ei_rope_table_scaled", None, *args)


@pytest.mark.parametrize("match,kw,rope_dim", [
    ("kind 4", dict(kind=4), 128),
    ("kind -1", dict(kind=-1), 128),
    ("factor 0.5", dict(kind=1, factor=0.5), 128),
    ("factor nan", dict(kind=1, factor=float("nan")), 128),
    ("factor inf", dict(kind=3, factor=float("inf")), 128),
    ("more than one pair", dict(kind=2, factor=2.0), 2),
    ("n_trained 0", dict(kind=3, factor=2.0, n_trained=0), 128),
    ("beta_fast", dict(kind=3, factor=2.0, beta_fast=0.5), 128),
    ("beta_fast", dict(kind=3, factor=2.0, beta_slow=0.0), 128),
    ("beta_fast", dict(kind=3, factor=2.0, beta_fast=float("nan")), 128),
    ("attn_factor", dict(kind=3, factor=2.0, attn_factor=float("inf")), 128),
])
def test_scaling_arguments(match, kw, rope_dim):
    _refused(match, "ei_rope_table_scaled", None, P, 16, rope_dim, 1e6, _scaling(**kw))


def _rope(**kw):
    d = dict(x=FAR[0], xs=4096, y=FAR[1], ys=4096, rows=8, n_heads=32, head_dim=128, gamma=None, eps=1e-6, cs=FAR[2],
             n_pos=64, pos=FAR[3], rope_dim=128, layout=0)
    d.update(kw)
    return (None, *d.values())


@pytest.mark.parametrize("match,kw", [
    ("head_dim 64", dict(head_dim=64)),
    ("rope_dim 130", dict(rope_dim=130)),
    ("rope_dim 3", dict(rope_dim=3)),
    ("layout 2", dict(layout=2)),
    ("null", dict(x=None)),
    ("null", dict(y=None)),
    ("null", dict(cs=None)),
    ("null", dict(pos=None)),
    ("rows -1", dict(rows=-1)),
    ("n_heads 0", dict(n_heads=0)),
    ("n_pos 0", dict(n_pos=0)),
    ("above 2\\^31", dict(rows=1 << 30, n_heads=4)),
    ("strides", dict(xs=4095)),
    ("strides", dict(xs=4098)),
    ("strides", dict(ys=4092)),
    ("aligned", dict(x=ctypes.c_void_p((2 << 40) + 4))),
    ("aligned", dict(gamma=_at(8))),
    ("overlaps", dict(y=ctypes.c_void_p((2 << 40) + 512))),
    ("overlaps", dict(y=FAR[0], ys=4100)),
    ("overlaps", dict(x=FAR[0], y=ctypes.c_void_p((2 << 40) - 16))),
])
def test_rope_rows_arguments(match, kw):
    _refused(match, "ei_rope_rows", *_rope(**kw))


def test_nothing_to_do_is_no_error():
    from exactinfer_amd import _capi
    _capi.call("ei_rope_rows", *_rope(rows=0))
    _capi.call("ei_attn_packed", *_packed(rows=0))
    _capi.call("ei_attn_packed_paged", *_paged(rows=0))
    _capi.call("ei_packed_step_paged", *_step(rows=0))


def test_sizes():
    from exactinfer_amd import _capi
    L = _capi.lib()
    assert L.ei_packed_plan_bytes(4, 100, 32, 8) > 0 and L.ei_packed_ws_bytes(100, 32, 8) > 0
    assert L.ei_packed_plan_bytes(1, 0, 8, 8) > 0
    for bad in ((0, 100, 32, 8), (65536, 100, 32, 8), (4, -1, 32, 8), (4, (1 << 20) + 1, 32, 8), (4, 100, 30, 8),
                (4, 100, 128, 8), (4, 100, 0, 8), (4, 100, 32, 0), (4, 100, 4096, 2048), (4, 1 << 20, 512, 64)):
        assert L.ei_packed_plan_bytes(*bad) == 0, bad
        if bad[0] == 4:
            assert L.ei_packed_ws_bytes(*bad[1:]) == 0, bad
    # the sizes grow with every argument: one buffer serves every smaller batch
    last = 0
    for n_seq, rows in ((1, 1), (3, 1), (3, 50), (40, 50), (40, 3000), (65535, 1 << 18)):
        now = L.ei_packed_plan_bytes(n_seq, rows, 40, 8)
        assert now >= last
        last = now


@pytest.mark.parametrize("match,args", [
    ("GQA group 16", (P, None, 4, 100, 100, 128, 8, P, BIG)),
    ("multiple", (P, None, 4, 100, 100, 30, 8, P, BIG)),
    ("n_seq 0", (P, None, 0, 100, 100, 32, 8, P, BIG)),
    ("n_seq 65536", (P, None, 65536, 100, 100, 32, 8, P, BIG)),
    ("rows -1", (P, None, 4, -1, 100, 32, 8, P, BIG)),
    ("2\\^20 rows", (P, None, 4, (1 << 20) + 1, 100, 32, 8, P, BIG)),
    ("max_kv -1", (P, None, 4, 100, -1, 32, 8, P, BIG)),
    ("max_kv", (P, None, 4, 100, (1 << 30) + 1, 32, 8, P, BIG)),
    ("cu_rows", (None, None, 4, 100, 100, 32, 8, P, BIG)),
    ("plan missing", (P, None, 4, 100, 100, 32, 8, None, BIG)),
    ("ei_packed_plan_bytes", (P, None, 4, 100, 100, 32, 8, P, 64)),
    ("aligned", (P, None, 4, 100, 100, 32, 8, _at(8), BIG)),
])
def test_plan_arguments(match, args):
    _refused(match, "ei_packed_plan", None, *args)


def _packed(**kw):
    d = dict(q=FAR[0], qs=6144, k=_off(FAR[0], 4096), v=_off(FAR[0], 5120), kvs=6144, out=FAR[1], n_seq=4, rows=100,
             H=32, HKV=8, D=128, scale=0.1, plan=FAR[2], pb=BIG, ws=FAR[3], wb=BIG)
    d.update(kw)
    return (None, *d.values())


def _off(p, floats):
    return ctypes.c_void_p(p.value + 4 * floats)


def _paged(**kw):
    d = dict(q=FAR[0], qs=6144, out=FAR[1], kc=FAR[4], vc=FAR[5], n_blocks=10, table=FAR[6], max_blocks=4, bs=64,
             n_seq=4, rows=100, H=32, HKV=8, D=128, scale=0.1, plan=FAR[2], pb=BIG, ws=FAR[3], wb=BIG)
    d.update(kw)
    return (None, *d.values())


def _step(**kw):
    d = dict(qkv=FAR[0], rs=6144, out=FAR[1], kc=FAR[4], vc=FAR[5], n_blocks=10, table=FAR[6], max_blocks=4, bs=64,
             n_seq=4, rows=100, H=32, HKV=8, D=128, qg=P, kg=P, cs=FAR[7], n_pos=64, rope_dim=128, eps=1e-6, scale=0.1,
             plan=FAR[2], pb=BIG, ws=FAR[3], wb=BIG)
    d.update(kw)
    return (None, *d.values())


COMMON = [
    ("head_dim 64", dict(D=64)),
    ("GQA group 16", dict(H=128)),
    ("multiple", dict(H=30)),
    ("n_seq 0", dict(n_seq=0)),
    ("rows -1", dict(rows=-1)),
    ("2\\^20 rows", dict(rows=(1 << 20) + 1)),
    ("plan missing", dict(plan=None)),
    ("ei_packed_plan_bytes", dict(pb=100)),
    ("ei_packed_ws_bytes", dict(wb=100)),
    ("workspace missing", dict(ws=None)),
    ("out missing", dict(out=None)),
    ("out missing", dict(out=_off(FAR[1], 1))),
    ("overlap", dict(ws=FAR[1])),
    ("overlap", dict(plan=FAR[1])),
    ("overlap", dict(plan=FAR[3])),
]
POOL = [
    ("block_size 16", dict(bs=16)),
    ("block_size 48", dict(bs=48)),
    ("block_size 0", dict(bs=0)),
    ("max_blocks 0", dict(max_blocks=0)),
    ("2\\^31", dict(max_blocks=1 << 26)),
    ("n_blocks 0", dict(n_blocks=0)),
    ("null", dict(kc=None)),
    ("null", dict(vc=None)),
    ("null", dict(table=None)),
    ("aligned", dict(kc=_off(FAR[4], 1))),
    ("lies in a pool", dict(kc=_off(FAR[1], 4096))),
    ("lies in a pool", dict(vc=_off(FAR[3], 4096))),
]


@pytest.mark.parametrize("match,kw", COMMON + [
    ("null", dict(q=None)),
    ("null", dict(k=None)),
    ("aligned", dict(v=_off(FAR[0], 5121))),
    ("q_stride", dict(qs=4092)),
    ("q_stride", dict(qs=6145)),
    ("kv_stride", dict(kvs=1020)),
    ("kv_stride", dict(kvs=6146)),
    ("kv_stride", dict(kvs=1 << 23)),
    ("overlaps q", dict(out=_off(FAR[0], 6144))),
    ("overlaps q", dict(out=FAR[5], k=FAR[5])),
    ("overlaps q", dict(out=FAR[5], v=_off(FAR[5], 4096))),
    ("workspace overlaps", dict(ws=_off(FAR[0], 4096))),
    ("workspace overlaps", dict(ws=FAR[5], k=FAR[5])),
    ("workspace overlaps", dict(ws=FAR[5], v=FAR[5])),
])
def test_packed_arguments(match, kw):
    _refused(match, "ei_attn_packed", *_packed(**kw))


@pytest.mark.parametrize("match,kw", COMMON + POOL + [
    ("q missing", dict(q=None)),
    ("q_stride", dict(qs=4092)),
    ("overlaps q", dict(out=_off(FAR[0], 4096))),
    ("workspace overlaps", dict(ws=_off(FAR[0], 4096))),
])
def test_paged_arguments(match, kw):
    _refused(match, "ei_attn_packed_paged", *_paged(**kw))


@pytest.mark.parametrize("match,kw", COMMON + POOL + [
    ("null", dict(qkv=None)),
    ("null", dict(qg=None)),
    ("null", dict(kg=None)),
    ("null", dict(cs=None)),
    ("n_pos 0", dict(n_pos=0)),
    ("rope_dim 5", dict(rope_dim=5)),
    ("row_stride", dict(rs=6140)),
    ("row_stride", dict(rs=6146)),
    ("overlaps qkv", dict(out=FAR[0])),
    ("overlaps qkv", dict(ws=_off(FAR[0], 6144))),
    ("qkv lies in a pool", dict(vc=_off(FAR[0], 4096))),
    ("pools overlap", dict(vc=_off(FAR[4], 1024))),
])
def test_step_arguments(match, kw):
    _refused(match, "ei_packed_step_paged", *_step(**kw))


@pytest.mark.parametrize("kw", [
    dict(cs=_off(FAR[1], 8 * 4096 - 4)), dict(cs=ctypes.c_void_p(FAR[1].value - 64 * 128 * 4 + 16)),
    dict(pos=_off(FAR[1], 4096)), dict(pos=ctypes.c_void_p(FAR[1].value - 8 * 4 + 4)),
    dict(gamma=_off(FAR[1], 512)), dict(y=FAR[0], gamma=_off(FAR[0], 128)), dict(y=FAR[0], cs=FAR[0]),
])
def test_rope_rows_over_its_own_tables(kw):
    """Rows that would be written over the table, the positions or gamma, which other rows still read."""
    _refused("overlaps cs, pos or gamma", "ei_rope_rows", *_rope(**kw))


@pytest.mark.parametrize("cu,kv", [(_at(0), None), (_at(-16), None), (FAR[0], _at(256)), (FAR[0], _at(-12))])
def test_plan_over_its_lengths(cu, kv):
    """The plan is written while its workgroup reads them."""
    _refused("plan overlaps", "ei_packed_plan", None, cu, kv, 4, 100, 100, 32, 8, P, BIG)


@pytest.mark.parametrize("at", ["out", "ws"])
def test_paged_table_that_the_call_writes(at):
    for call, args in (("ei_attn_packed_paged", _paged), ("ei_packed_step_paged", _step)):
        to = {"out": FAR[1], "ws": FAR[3]}[at]
        _refused("overlaps the block table", call, *args(table=_off(to, 1024)))
        _refused("overlaps the block table", call, *args(table=ctypes.c_void_p(to.value - 4 * 4 * 4 + 4)))


@pytest.mark.parametrize("what", ["plan", "table", "qg", "kg", "cs"])
@pytest.mark.parametrize("into", ["kc", "vc", "out", "ws"])
def test_step_inputs_that_it_writes(what, into):
    """What the step reads must not lie in the pools, the outputs or the workspace."""
    to = dict(kc=FAR[4], vc=FAR[5], out=FAR[1], ws=FAR[3])[into]
    _refused("overlap", "ei_packed_step_paged", *_step(**{what: _off(to, 4096)}))
    _refused("overlap", "ei_packed_step_paged", *_step(**{what: ctypes.c_void_p(to.value - 16)}))
