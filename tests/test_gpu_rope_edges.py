"""GPU tests of rotary positions (include/ei_packed.h) at the edges of their arguments."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def test_rows_side_by_side_in_one_buffer(gpu):
    """Columns of one buffer turned into other columns of it: the rows lie between each other and share nothing."""
    rows, H = 37, 4
    g = torch.Generator(device="cuda").manual_seed(301)
    buf = torch.randn((rows, 3 * H * D + 8), generator=g, device="cuda")
    cs = gpu.rope_table_scaled(64)
    pos = torch.randint(0, 64, (rows,), generator=g, device="cuda", dtype=torch.int32)
    want = gpu.rope_rows(buf[:, H * D:2 * H * D], H, cs, pos)
    for x, y in ((1, 2), (1, 0)):
        b = buf.clone()
        gpu.rope_rows(b[:, x * H * D:(x + 1) * H * D], H, cs, pos, out=b[:, y * H * D:(y + 1) * H * D])
        assert torch.equal(b[:, y * H * D:(y + 1) * H * D], want)
        b[:, y * H * D:(y + 1) * H * D] = buf[:, y * H * D:(y + 1) * H * D]
        assert torch.equal(b, buf)
    # four values into the other's columns, before and behind them, and from a row's end into the next row
    for x, y in ((0, H * D - 4), (H * D - 4, 0), (2 * H * D + 12, 0), (0, 2 * H * D + 12)):
        a, b = (buf.as_strided((rows - 1, H * D), buf.stride(), at) for at in (x, y))
        with pytest.raises(RuntimeError, match="overlaps"):
            gpu.rope_rows(a, H, cs, pos[1:], out=b)


@pytest.mark.parametrize("n_trained,beta_slow", [(4, 1.0), (6, 1.0), (100, 16.0)])
def test_yarn_where_no_pair_is_fast(gpu, n_trained, beta_slow):
    """Every pair makes at most beta_slow turns over the trained positions: all of them are slowed by factor."""
    yarn = gpu.RopeScaling("yarn", 4.0, n_trained, 32.0, beta_slow, 1.0)
    assert n_trained / (2 * np.pi) <= beta_slow
    assert torch.equal(gpu.rope_table_scaled(300, scaling=yarn),
                       gpu.rope_table_scaled(300, scaling=gpu.RopeScaling("linear", 4.0)))
