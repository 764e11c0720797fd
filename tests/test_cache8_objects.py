"""Cache8 objects: what a call is told about the pool is what the object's tensors are then."""
import pytest
import torch

from exactinfer_amd import attention as A


def _cache(kind="int8", device="cpu"):
    return A.Cache8(3, 32, 2, kind, device=device)


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "kind", "n_blocks", "n_head_kv", "block_size"])
def test_what_a_pool_is_made_of_cannot_be_assigned(name):
    c = _cache()
    with pytest.raises(AttributeError):
        setattr(c, name, getattr(c, name))


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_addresses_are_those_at_the_call(name):
    c = _cache()
    t = getattr(c, name)
    t.data = torch.ones_like(t)  # (another storage under the same tensor, as moving a module's buffers does)
    c._address()
    assert getattr(c._c, name) == t.data_ptr()


def test_other_shapes_under_the_same_tensors():
    c = _cache()
    for name in ("k", "v", "k_scale", "v_scale"):
        t = getattr(c, name)
        t.data = torch.ones((2, *t.shape[1:]), dtype=t.dtype)
    c._address()
    assert c._c.n_blocks == c.n_blocks == 2
    c.v.data = torch.ones((5, 2, 32, 128), dtype=torch.int8)
    with pytest.raises(ValueError, match="v must be"):
        c._address()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_calls_follow_the_tensors(gpu, kind):
    from tests.cache8_plain import D, Batch, fill_cache
    b = Batch(gpu, 8, 4, [1, 5], [70, 40], 32, seed=1)
    one, two = (fill_cache(gpu, kind, b.n_blocks, 32, 4, seed) for seed in (2, 3))
    q = torch.randn((b.rows, 8 * D), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    old = gpu.attn_packed_cache8(q, one, b.table, b.plan, b.shape)
    want = gpu.attn_packed_cache8(q, two, b.table, b.plan, b.shape)
    kept = [t.data for t in (one.k, one.v, one.k_scale, one.v_scale)]  # (the old storage stays)
    for x, y in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        x.data = y.data
    got = gpu.attn_packed_cache8(q, one, b.table, b.plan, b.shape)
    assert torch.equal(got, want) and not torch.equal(got, old) and len(kept) == 4
