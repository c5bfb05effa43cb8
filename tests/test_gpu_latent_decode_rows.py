"""The paged latents' decode on each of its kernels -- up to 32 rows of q, up to
64, more, and widths that are no whole chunks -- where hidden rows are not finite
and where a split is longer than the table of places that a workgroup keeps."""
import math

import pytest
import torch

from attn_cases import DTYPES, near
from test_gpu_latent_decode import exact, make, run

pytestmark = pytest.mark.gpu
both = pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())


def without_page_0(table, count):
    """The table with another page in page 0's place, and the pages that it does not use, 0 among them."""
    unused = set(range(count)) - set(table.flatten().tolist())
    if 0 not in unused:
        other = max(unused)
        table[table == 0] = other
        unused = unused - {other} | {0}
    return table, sorted(unused)


@both
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("H,d_c,d_r", [(8, 128, 16), (8, 256, 64), (8, 512, 64), (10, 128, 16), (10, 256, 64), (10, 512, 64),
                                       (30, 128, 16), (30, 256, 0), (30, 512, 64), (8, 101, 7), (30, 500, 3)])
def test_hidden_rows_have_no_part(device, dtype, value, H, d_c, d_r):
    """Pages that no sequence has, rows behind a length, rows that only the last
    steps see, and row 0, which stands in for rows of pages that are not there."""
    lens, steps, page = [45, 300, 1300], 4, 32
    q, cache, table, n = make(lens, steps, H, d_c, d_r, page, dtype, seed=21)
    table, unused = without_page_0(table, cache.shape[0])
    assert 0 in unused and len(unused) == 3 and not bool((table == 0).any())
    table[1, 3] = -1
    table[2, 20] = cache.shape[0]
    want, tol = exact(q, cache, table, n, d_c, 0.06, dtype, page)
    assert bool(torch.isfinite(want[0]).all())
    for i in unused:
        cache[i] = value
    for b, length in enumerate(lens):
        cache[table[b, length // page], length % page:] = value
    got = run(q, cache, table, n, d_c, 0.06, device)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")
    for b, length in enumerate(lens):  # what the last two steps see
        cache[table[b, (length - 2) // page], (length - 2) % page, d_c // 2] = value
    got = run(q, cache, table, n, d_c, 0.06, device)
    near(got[0][:, :2], want[0][:, :2], tol[0][:, :2], "o of the earlier steps")
    near(got[1][:, :2], want[1][:, :2], tol[1][:, :2], "lse of the earlier steps")
    if math.isnan(value):
        assert bool(torch.isnan(got[0][:, 2:]).all()) and bool(torch.isnan(got[1][:, 2:]).all())


@both
@pytest.mark.parametrize("steps,H,d_c", [(1, 2, 32), (4, 10, 32), (16, 8, 32), (1, 2, 33), (4, 10, 33)])
def test_splits_longer_than_the_table_of_places(device, dtype, steps, H, d_c):
    """140000 positions are 125 splits of 1120 (the table has 1024), and 2500 beside them a few."""
    n = [140000, 2500]
    q, cache, table, lens = make(n, steps, H, d_c, 0, 128, dtype, seed=22)
    got = run(q, cache, table, lens, d_c, 0.2, device)
    want, tol = exact(q, cache, table, lens, d_c, 0.2, dtype, 128)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")


@both
@pytest.mark.parametrize("H", [8, 40, 100])
@pytest.mark.parametrize("length", [40, 2000])
def test_values_near_the_largest(device, dtype, H, length):
    """Latents whose sum over some hundred rows leaves fp32's range, and whose mean does not."""
    q, cache, table, n = make([length], 1, H, 128, 16, 64, dtype, seed=23)
    cache[..., 5], q[..., 5] = 1.5e37, 0.0
    cache[..., 6], q[..., 6] = 1e36 * cache[..., 6], 0.0
    got = run(q, cache, table, n, 128, 0.05, device)
    want, tol = exact(q, cache, table, n, 128, 0.05, dtype, 64)
    near(got[0], want[0], tol[0], "o")
    near(got[1], want[1], tol[1], "lse")
