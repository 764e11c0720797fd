"""GPU tests of the rotary operators (ei_rope_table_scaled, ei_rope_rows) against 64-bit forms.

Tolerances.  u = 2^-24 is half a step of fp32.  A table entry is rounded once (u of its size, plus the
double-precision angle's error, 2^-53 of up to 2^17 radians: far below u).  A turned value a c - b s
takes, per product, the table's u and its own u, and u of the sum; with the norm first, a and b
carry inv's, the product's and gamma's u each (3u): (2 + 3) u (|a c| + |b s|) + u |sum| <=
5 sqrt(2) u r + u r < 8.1 u r, r the pair's length (times m, the table's factor).  Second-order terms
are below 2^-40 r, so 8.2 u r with the norm; without it 2 sqrt(2) u r + u r < 3.9 u r.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
U = 2.0 ** -24
KINDS = ["none", "linear", "ntk", "yarn"]


def _frequencies(rd, theta, kind, factor=1.0, trained=0, fast=32.0, slow=1.0, attn=0.0):
    i = np.arange(rd // 2, dtype=np.float64)
    m = 1.0
    if kind == "ntk":
        theta = theta * factor ** (rd / (rd - 2))
    f = theta ** (-2.0 * i / rd)
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        turns = trained * f / (2 * math.pi)  # of each pair over the trained positions
        # the ramp runs over the pair index, between the (real) pairs that make `fast` and `slow` turns
        at = [rd / 2 * math.log(trained / (2 * math.pi * n)) / math.log(theta) for n in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rd - 1)
        share = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        assert np.all(share[turns > fast * theta ** (2 / rd)] == 0) or lo == 0
        f = f * (1 - share) + f / factor * share
        m = attn if attn > 0 else 0.1 * math.log(factor) + 1
    return f, m


def _turn64(x, pos, f, m, rd, layout, gamma=None, eps=1e-6):
    """x [rows, heads, 128] in 64 bits; returns it turned and each value's pair length."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma if gamma is not None else x.copy()
    out, size = y.copy(), np.abs(y)
    th = pos[:, None].astype(np.float64) * f
    c, s = m * np.cos(th)[:, None], m * np.sin(th)[:, None]
    ia = np.arange(rd // 2) if layout == "half" else 2 * np.arange(rd // 2)
    ib = ia + (rd // 2 if layout == "half" else 1)
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = m * np.hypot(a, b)
    return out, size


@pytest.mark.parametrize("rd", [2, 10, 64, 96, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_table(gpu, kind, rd):
    if kind == "ntk" and rd == 2:
        pytest.skip("one pair: refused")
    n, theta = 40000, 1e6
    cs = gpu.rope_table_scaled(n, rd, theta, gpu.RopeScaling(kind, 4.0, 8192)).cpu().numpy()
    f, m = _frequencies(rd, theta, kind, 4.0, 8192)
    p = np.concatenate([np.arange(300), np.arange(n - 300, n), np.arange(0, n, 997)])
    th = p[:, None] * f
    # the angle p f_i is off by a few 2^-53 of itself (pow, product): at most 40000 * 2^-50
    tol = U * m + 40000 * 2.0 ** -50
    assert np.abs(cs[p, :, 0] - m * np.cos(th)).max() <= tol
    assert np.abs(cs[p, :, 1] - m * np.sin(th)).max() <= tol


def test_table_without_scaling_is_the_host_table(gpu):
    """Rounded from the same doubles: where the two differ it is by one step, at a rounding tie."""
    a, b = gpu.rope_table(2048).cpu().numpy(), gpu.rope_table_scaled(2048).cpu().numpy()
    assert np.mean(a.view(np.int32) != b.view(np.int32)) < 1e-5
    assert np.abs(a - b).max() <= 2 * U


def test_yarn_factors(gpu):
    sc = gpu.RopeScaling("yarn", 2.5, 1000, beta_fast=20.0, beta_slow=2.0, attn_factor=1.25)
    cs = gpu.rope_table_scaled(50, 128, 1e4, sc).cpu().numpy()
    f, m = _frequencies(128, 1e4, "yarn", 2.5, 1000, 20.0, 2.0, 1.25)
    assert m == 1.25
    assert np.abs(cs[:, :, 0] - m * np.cos(np.arange(50)[:, None] * f)).max() <= 2 * U


CASES = [  # rows, heads, extra columns, rope_dim
    (1, 1, 0, 128), (3, 5, 0, 128), (37, 10, 256, 128), (200, 40, 1024, 128), (64, 16, 4, 64), (33, 9, 0, 96),
    (17, 3, 128, 2), (5, 7, 0, 4), (40, 6, 0, 10), (21, 4, 12, 90), (700, 2, 0, 126), (1, 33, 0, 32),
]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rows,heads,extra,rd", CASES)
def test_rows(gpu, rows, heads, extra, rd, norm, layout):
    rng = np.random.default_rng(rows * 1000 + rd)
    n_pos, width = 5000, heads * D
    x = rng.standard_normal((rows, width + extra)).astype(np.float32)
    pos = rng.integers(0, n_pos, rows).astype(np.int32)
    pos[rng.integers(0, rows)] = n_pos - 1
    gamma = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32) if norm else None
    cs = gpu.rope_table_scaled(n_pos, rd, 1e4)
    f, m = _frequencies(rd, 1e4, "none")
    xd = torch.from_numpy(x).cuda()
    args = (heads, cs, torch.from_numpy(pos).cuda())
    kw = dict(rope_dim=rd, layout=layout, gamma=None if gamma is None else torch.from_numpy(gamma).cuda())
    ref, size = _turn64(x[:, :width].astype(np.float64).reshape(rows, heads, D), pos, f, m, rd, layout, gamma)
    tol = (8.2 if norm else 3.9) * U * size
    # out of place, into rows of another stride whose other columns stay as they are
    out = torch.full((rows, width + 8), 7.0, device="cuda")
    gpu.rope_rows(xd, *args, out=out, **kw)
    o = out.cpu().numpy()
    err = np.abs(o[:, :width].reshape(rows, heads, D) - ref)
    assert np.all(err <= tol), (err / np.maximum(size, 1e-30)).max() / U
    assert np.all(o[:, width:] == 7.0) and np.array_equal(xd.cpu().numpy(), x)
    # in place: the same bits, other columns untouched
    gpu.rope_rows(xd, *args, out=xd, **kw)
    got = xd.cpu().numpy()
    assert np.array_equal(got[:, :width], o[:, :width]) and np.array_equal(got[:, width:], x[:, width:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rd", [128, 64, 10])
def test_rows_outside_the_table_are_copied(gpu, rd, norm, layout):
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((6, 3 * D)).astype(np.float32)).cuda()
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    pos = torch.tensor([4, -1, 64, 63, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    cs = gpu.rope_table_scaled(64, rd)
    gamma = torch.full((D,), 1.5, device="cuda") if norm else None
    out = gpu.rope_rows(x, 3, cs, pos, rope_dim=rd, layout=layout, gamma=gamma)
    for r in (1, 2, 4, 5):
        assert torch.equal(out[r].view(torch.int32), x[r].view(torch.int32)), r
    for r in (0, 3):
        assert not torch.equal(out[r], x[r]) and torch.isfinite(out[r]).all()


def test_same_as_the_chunk_prologue(gpu):
    """Rows at consecutive positions: the values of ei_headnorm_rope, but for a last bit where the sums of
    squares, added in another order, round to neighbouring factors."""
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((50, 8 * D)).astype(np.float32)).cuda()
    gamma = torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).cuda()
    cs = gpu.rope_table(400)
    pos = torch.arange(300, 350, dtype=torch.int32, device="cuda")
    got = gpu.rope_rows(x, 8, cs, pos, gamma=gamma)
    ref = x.clone()
    gpu.headnorm_rope(ref, 8, gamma, cs, torch.tensor([300], dtype=torch.int32, device="cuda"))
    same = (got == ref).float().mean().item()
    assert same > 0.999 and (got - ref).abs().max().item() <= 2 ** -21


def test_many_rows_and_far_positions(gpu):
    """More rows than one round of workgroups takes, the last positions of a long table."""
    rows, heads, n_pos = 9001, 3, 131072
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((rows, heads * D), generator=g, device="cuda")
    pos = torch.randint(n_pos - 500, n_pos, (rows,), generator=g, device="cuda", dtype=torch.int32)
    sc = gpu.RopeScaling("yarn", 4.0, 32768)
    cs = gpu.rope_table_scaled(n_pos, D, 1e6, sc)
    out = gpu.rope_rows(x, heads, cs, pos, layout="interleaved").cpu().numpy()
    f, m = _frequencies(D, 1e6, "yarn", 4.0, 32768)
    ref, size = _turn64(x.cpu().numpy().astype(np.float64).reshape(rows, heads, D), pos.cpu().numpy(), f, m, D,
                        "interleaved")
    # (the angle itself is off by a few 2^-53 of 131072 radians)
    assert np.all(np.abs(out.reshape(ref.shape) - ref) <= (3.9 * U + 131072 * 2.0 ** -50) * size)


def test_python_refusals(gpu):
    x = torch.zeros((4, 2 * D), device="cuda")
    cs, pos = gpu.rope_table_scaled(16), torch.zeros(4, dtype=torch.int32, device="cuda")
    ok = dict(x=x, n_heads=2, cs=cs, pos=pos)
    for match, kw in (("layout", dict(layout="pairs")), ("int32", dict(pos=pos.long())), ("float32", dict(x=x.half())),
                      ("rows of", dict(n_heads=3)),
                      ("rows of", dict(pos=torch.zeros(5, dtype=torch.int32, device="cuda"))),
                     
                      ("cs must be", dict(rope_dim=64)), ("contiguous", dict(x=x.t())), ("GPU tensor", dict(x=x.cpu())),
                      ("128 values", dict(gamma=x[0])), ("rows of", dict(out=x[:3])),
                      ("overlaps", dict(x=x[:3], out=x[1:], pos=pos[:3]))):
        with pytest.raises((ValueError, RuntimeError), match=match):
            gpu.rope_rows(**{**ok, **kw})
    with pytest.raises(ValueError, match="scaling kind"):
        gpu.rope_table_scaled(16, scaling=gpu.RopeScaling("cubic"))
    assert gpu.rope_rows(x[:0], 2, cs, pos[:0]).shape == (0, 2 * D)
