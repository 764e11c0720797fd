"""Refusals of include/ei_cache8.h's entry points: every check that comes before a launch (CPU only)."""
import ctypes

import pytest
import torch

FAR = [ctypes.c_void_p((i + 2) << 40) for i in range(16)]  # addresses far apart; never dereferenced
BIG = 1 << 38


def _off(p, nbytes):
    return ctypes.c_void_p(p.value + nbytes)


def _cache(**kw):
    from exactinfer_amd import _capi
    d = dict(k=FAR[8], v=FAR[9], ks=FAR[10], vs=FAR[11], kind=1, n_blocks=10, bs=64)
    d.update({k: v for k, v in kw.items() if k in d})
    as_int = [d[k].value if isinstance(d[k], ctypes.c_void_p) else d[k] for k in ("k", "v", "ks", "vs")]
    c = _capi.Cache8C(*as_int, d["kind"], d["n_blocks"], d["bs"])
    return ctypes.byref(c)


_CACHE_KEYS = ("k", "v", "ks", "vs", "kind", "n_blocks", "bs")
CACHE8 = {
    "ei_cache8_store": dict(qkv=FAR[0], rs=6144, out=FAR[1], cache=None, table=FAR[6], max_blocks=4, n_seq=4, rows=100,
                            H=32, HKV=8, D=128, qg=FAR[12], kg=FAR[13], cs=FAR[7], n_pos=64, turn=FAR[14], rope_dim=128,
                            eps=1e-6, plan=FAR[2], pb=BIG),
    "ei_cache8_load": dict(cache=None, table=FAR[6], max_blocks=4, out=FAR[1], v_out=FAR[0], stride=1024, n_seq=4,
                           rows=100, H=32, HKV=8, D=128, plan=FAR[2], pb=BIG),
    "ei_attn_packed_cache8": dict(q=FAR[0], qs=6144, out=FAR[1], cache=None, table=FAR[6], max_blocks=4, n_seq=4,
                                  rows=100, H=32, HKV=8, D=128, mask=FAR[15], words=1, scale=0.1, plan=FAR[2], pb=BIG,
                                  ws=FAR[3], wb=BIG),
    "ei_packed_step_cache8": dict(qkv=FAR[0], rs=6144, out=FAR[1], cache=None, table=FAR[6], max_blocks=4, n_seq=4,
                                  rows=100, H=32, HKV=8, D=128, qg=FAR[12], kg=FAR[13], cs=FAR[7], n_pos=64,
                                  turn=FAR[14], rope_dim=128, eps=1e-6, mask=FAR[15], words=1, scale=0.1, plan=FAR[2],
                                  pb=BIG, ws=FAR[3], wb=BIG),
    "ei_cache8_keep": dict(cache=None, table=FAR[6], max_blocks=4, n_seq=4, rows=100, H=32, HKV=8, D=128, kept=FAR[0],
                           max_kept=9, n_kept=FAR[12], new_len=FAR[1], plan=FAR[2], pb=BIG),
}
POOL = {
    "ei_attn_tree_paged": dict(q=FAR[0], qs=6144, out=FAR[1], kc=FAR[4], vc=FAR[5], n_blocks=10, table=FAR[6],
                               max_blocks=4, bs=64, n_seq=4, rows=100, H=32, HKV=8, D=128, mask=FAR[15], words=1,
                               scale=0.1, plan=FAR[2], pb=BIG, ws=FAR[3], wb=BIG),
    "ei_tree_step_paged": dict(qkv=FAR[0], rs=6144, out=FAR[1], kc=FAR[4], vc=FAR[5], n_blocks=10, table=FAR[6],
                               max_blocks=4, bs=64, n_seq=4, rows=100, H=32, HKV=8, D=128, qg=FAR[12], kg=FAR[13],
                               cs=FAR[7], n_pos=64, turn=FAR[14], rope_dim=128, eps=1e-6, mask=FAR[15], words=1,
                               scale=0.1, plan=FAR[2], pb=BIG, ws=FAR[3], wb=BIG),
    "ei_cache_keep": dict(kc=FAR[4], vc=FAR[5], n_blocks=10, table=FAR[6], max_blocks=4, bs=64, n_seq=4, rows=100, H=32,
                          HKV=8, D=128, kept=FAR[0], max_kept=9, n_kept=FAR[12], new_len=FAR[1], plan=FAR[2], pb=BIG),
}
ALL = {**CACHE8, **POOL}


def _call(name, **kw):
    from exactinfer_amd import _capi
    d = dict(ALL[name])
    if name in CACHE8:
        given = kw.pop("cache", "made")
        d["cache"] = _cache(**kw) if given == "made" else given
        kw = {k: v for k, v in kw.items() if k not in _CACHE_KEYS}
    assert set(kw) <= set(d), (name, kw)
    d.update(kw)
    _capi.call(name, None, *d.values())


def _refused(match, name, **kw):
    from exactinfer_amd import _capi
    with pytest.raises(_capi.EiError, match=match):
        _call(name, **kw)


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("match,kw", [
    ("head_dim 64", dict(D=64)),
    ("GQA group 16", dict(H=128)),
    ("multiple", dict(H=30)),
    ("n_seq 0", dict(n_seq=0)),
    ("n_seq 65536", dict(n_seq=65536)),
    ("rows -1", dict(rows=-1)),
    ("2\\^20 rows", dict(rows=(1 << 20) + 1)),
    ("plan missing", dict(plan=None)),
    ("plan missing", dict(plan=_off(FAR[2], 8))),
    ("ei_packed_plan_bytes", dict(pb=100)),
    ("block_size 16", dict(bs=16)),
    ("block_size 48", dict(bs=48)),
    ("block_size 0", dict(bs=0)),
    ("max_blocks 0", dict(max_blocks=0)),
    ("2\\^31", dict(max_blocks=1 << 26)),
    ("n_blocks 0", dict(n_blocks=0)),
    ("null", dict(table=None)),
])
def test_batch_and_pages(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("name", CACHE8)
@pytest.mark.parametrize("match,kw", [
    ("null", dict(cache=None)),
    ("null", dict(k=None)),
    ("null", dict(v=None)),
    ("null", dict(ks=None)),
    ("null", dict(vs=None)),
    ("kind 0", dict(kind=0)),
    ("kind 3", dict(kind=3)),
    ("aligned", dict(k=_off(FAR[8], 8))),
    ("aligned", dict(vs=_off(FAR[11], 4))),
])
def test_cache(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("name", [n for n in ALL if "ws" in ALL[n]])
@pytest.mark.parametrize("match,kw", [
    ("workspace missing", dict(ws=None)),
    ("ei_packed_ws_bytes", dict(wb=100)),
    ("out missing", dict(out=None)),
    ("out missing", dict(out=_off(FAR[1], 4))),
    ("mask_words 0", dict(words=0)),
    ("mask_words -1", dict(words=-1)),
    ("mask must be 8-byte aligned", dict(mask=_off(FAR[15], 4))),
    ("out overlaps the workspace", dict(ws=FAR[1])),
    ("out overlaps the plan", dict(plan=FAR[1])),
    ("workspace overlaps the plan", dict(plan=FAR[3])),
    ("out overlaps the mask", dict(mask=_off(FAR[1], 64))),
    ("workspace overlaps the mask", dict(mask=_off(FAR[3], 64))),
    ("out overlaps the block table", dict(table=_off(FAR[1], 64))),
    ("workspace overlaps the block table", dict(table=_off(FAR[3], 64))),
])
def test_outputs_and_masks(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("name", ["ei_attn_packed_cache8", "ei_attn_tree_paged"])
@pytest.mark.parametrize("match,kw", [
    ("q missing", dict(q=None)),
    ("q missing", dict(q=_off(FAR[0], 4))),
    ("q_stride", dict(qs=4092)),
    ("q_stride", dict(qs=6145)),
    ("out overlaps q", dict(out=_off(FAR[0], 16384))),
    ("workspace overlaps q", dict(ws=_off(FAR[0], 16384))),
])
def test_queries(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("name", [n for n in ALL if "qkv" in ALL[n]])
@pytest.mark.parametrize("match,kw", [
    ("null", dict(qkv=None)),
    ("null", dict(qg=None)),
    ("null", dict(kg=None)),
    ("null", dict(cs=None)),
    ("n_pos 0", dict(n_pos=0)),
    ("rope_dim 5", dict(rope_dim=5)),
    ("rope_dim 130", dict(rope_dim=130)),
    ("row_stride", dict(rs=6140)),
    ("row_stride", dict(rs=6146)),
    ("aligned", dict(qkv=_off(FAR[0], 4))),
    ("overlaps qkv", dict(out=FAR[0])),
    ("overlaps turn_at", dict(turn=_off(FAR[1], 64))),
    ("overlaps cs", dict(cs=_off(FAR[1], 64))),
    ("overlaps q_gamma", dict(qg=_off(FAR[1], 64))),
    ("overlaps k_gamma", dict(kg=_off(FAR[1], 64))),
    ("overlaps the plan", dict(plan=FAR[1])),
])
def test_raw_rows(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("what", ["qkv", "table", "plan", "turn", "qg", "kg", "cs"])
@pytest.mark.parametrize("into", ["k", "v", "ks", "vs"])
@pytest.mark.parametrize("name", ["ei_cache8_store", "ei_packed_step_cache8"])
def test_inputs_in_the_pool_that_is_written(name, what, into):
    to = dict(k=FAR[8], v=FAR[9], ks=FAR[10], vs=FAR[11])[into]
    _refused("overlaps", name, **{what: _off(to, 64)})


@pytest.mark.parametrize("what", ["qkv", "table", "plan", "turn", "qg", "kg", "cs", "mask"])
@pytest.mark.parametrize("into", [FAR[4], FAR[5]])
def test_inputs_in_the_fp32_pool_that_is_written(what, into):
    _refused("overlaps", "ei_tree_step_paged", **{what: _off(into, 64)})


@pytest.mark.parametrize("a,b", [("k", "v"), ("k", "ks"), ("k", "vs"), ("v", "ks"), ("v", "vs"), ("ks", "vs")])
@pytest.mark.parametrize("name", ["ei_cache8_store", "ei_packed_step_cache8", "ei_cache8_keep"])
def test_pool_over_itself(name, a, b):
    at = dict(k=FAR[8], v=FAR[9], ks=FAR[10], vs=FAR[11])[a]
    _refused("overlaps", name, **{b: _off(at, 128)})


@pytest.mark.parametrize("name", ["ei_tree_step_paged", "ei_cache_keep"])
def test_fp32_pools(name):
    _refused("overlaps", name, vc=_off(FAR[4], 4096))
    _refused("null", name, kc=None)
    _refused("null", name, vc=None)
    _refused("aligned", name, kc=_off(FAR[4], 4))


@pytest.mark.parametrize("out", ["out", "ws"])
@pytest.mark.parametrize("name,pools", [("ei_attn_packed_cache8", ("k", "v", "ks", "vs")),
                                        ("ei_packed_step_cache8", ("k", "v", "ks", "vs")),
                                        ("ei_attn_tree_paged", ("kc", "vc")), ("ei_tree_step_paged", ("kc", "vc"))])
def test_outputs_in_a_pool(name, pools, out):
    to = dict(out=FAR[1], ws=FAR[3])[out]
    for p in pools:
        _refused("overlaps", name, **{p: _off(to, 256)})


@pytest.mark.parametrize("match,kw", [
    ("missing", dict(out=None)),
    ("missing", dict(v_out=None)),
    ("missing", dict(out=_off(FAR[1], 4))),
    ("out_stride", dict(stride=1020)),
    ("out_stride", dict(stride=1026)),
    ("k_out overlaps v_out", dict(v_out=_off(FAR[1], 512))),
    ("k_out overlaps v_out", dict(v_out=FAR[1])),
    ("overlaps the K codes", dict(out=_off(FAR[8], 64))),
    ("overlaps the V scales", dict(v_out=_off(FAR[11], 64))),
    ("overlaps the block table", dict(v_out=FAR[6])),
    ("overlaps the plan", dict(out=FAR[2])),
])
def test_load_arguments(match, kw):
    _refused(match, "ei_cache8_load", **kw)


@pytest.mark.parametrize("name", ["ei_cache_keep", "ei_cache8_keep"])
@pytest.mark.parametrize("match,kw", [
    ("null", dict(kept=None)),
    ("null", dict(n_kept=None)),
    ("null", dict(new_len=None)),
    ("max_kept 0", dict(max_kept=0)),
    ("max_kept", dict(max_kept=(1 << 20) + 1)),
    ("overlaps kept", dict(new_len=_off(FAR[0], 16))),
    ("overlaps n_kept", dict(new_len=_off(FAR[12], 4))),
    ("overlaps the plan", dict(new_len=_off(FAR[2], 256))),
    ("overlaps the block table", dict(new_len=FAR[6])),
])
def test_keep_arguments(name, match, kw):
    _refused(match, name, **kw)


@pytest.mark.parametrize("what", ["kept", "n_kept", "new_len", "table", "plan"])
def test_keep_lists_in_a_pool(what):
    for p in (FAR[8], FAR[9], FAR[10], FAR[11]):
        _refused("overlaps", "ei_cache8_keep", **{what: _off(p, 64)})
    for p in (FAR[4], FAR[5]):
        _refused("overlaps", "ei_cache_keep", **{what: _off(p, 64)})


@pytest.mark.parametrize("name", [n for n in ALL if "keep" not in n])
def test_nothing_to_do_is_no_error(name):
    _call(name, rows=0)


def test_load_takes_columns_of_one_buffer():
    _call("ei_cache8_load", rows=0, out=FAR[1], v_out=_off(FAR[1], 4096), stride=2048)
    _refused("overlaps the plan", "ei_cache8_load", out=FAR[1], v_out=_off(FAR[1], 4096), stride=2048, plan=FAR[1])


def test_cache_objects():
    from exactinfer_amd import attention as A
    c = A.Cache8(3, 32, 2, "int8", device="cpu")
    assert c.k.shape == (3, 2, 32, 128) and c.k.dtype == torch.int8 and c.v_scale.shape == (3, 2, 32)
    assert A.Cache8.of(c.k, c.v, c.k_scale, c.v_scale).block_size == 32
    with pytest.raises(ValueError, match="kind"):
        A.Cache8(3, 32, 2, "int4", device="cpu")
    with pytest.raises(ValueError, match="float8_e4m3fn or torch.int8"):
        A.Cache8.of(c.k.float(), c.v, c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="v must be"):
        A.Cache8.of(c.k, c.v.view(torch.float8_e4m3fn), c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="k_scale must be"):
        A.Cache8.of(c.k, c.v, c.k_scale[:2], c.v_scale)
    with pytest.raises(ValueError, match="k must be|codes must be"):
        A.Cache8.of(c.k.transpose(1, 2), c.v, c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="codes must be"):
        A.Cache8.of(c.k[..., :64], c.v, c.k_scale, c.v_scale)
