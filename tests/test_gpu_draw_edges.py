"""GPU tests of lrs_draw_device at the ends of its definition, against draw_ref.py: uniforms that fall on a
step of the distribution function."""
import numpy as np
import pytest

import lrs
from test_gpu_draw import check, records, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiles,period,rows", [(128, 2, 64), (128, 2, 320), (149, 3, 64), (64, 2, 64), (40, 4, 16)])
@pytest.mark.parametrize("filters", [(1.0, 0, 1.0, 0.0), (1.0, 30000, 1.0, 0.0), (1.0, 0, 0.96875, 0.0)])
def test_uniforms_on_the_steps_between_closed_tiles(tiles, period, rows, filters):
    """Tiles of 1024 elements with the same values in each open one and nothing in the others, and uniforms j /
    64, which fall on the steps between tiles: there the sums of 64 bits decide by their last bit, so either
    neighbour of the step (1e-13 of the mass around it) is right, but never a closed element or none."""
    import torch
    rng = np.random.default_rng([tiles, period, rows])
    n = tiles * 1024
    one = rng.standard_normal(1024)
    x = np.where(np.arange(n) // 1024 % period == period - 1, np.tile(one, tiles), -np.inf).astype(np.float32)
    params = records(rows, [filters])
    u = (np.arange(rows) % 64 / 64).astype(np.float32)
    tok, prob, kept, status = run(torch.from_numpy(x[None]).cuda(), params, u, ld=0)
    assert (status == 0).all()
    w = np.exp(x.astype(np.float64) - x.max())
    order = np.argsort(-x, kind="stable")
    keep = int(np.isfinite(x).sum()) if filters[1] == 0 else min(filters[1], int(np.isfinite(x).sum()))
    if filters[2] < 1:
        keep = int((np.cumsum(w[order]) < filters[2] * w.sum()).sum()) + 1
        assert (np.abs(kept.astype(np.int64) - keep) <= 1).all()  # (top_p is on such a step as well)
    else:
        assert (kept == keep).all()
    k = np.zeros(n)
    k[order[:keep]] = w[order[:keep]]
    c = np.cumsum(k)
    # (the mass of one element is below 2^-14 of the whole; where the kept count is one off, so is the whole)
    off = c[-1] * 1e-13 + (k[order[keep - 1]] * 2 if filters[2] < 1 else 0.0)
    target = u.astype(np.float64) * c[-1]
    assert (tok < n).all()
    assert (k[tok] > 0).all()
    assert (c[tok] >= target - off).all() and (c[tok] - k[tok] <= target + off).all()
    assert (np.abs(prob - k[tok] / c[-1]) <= k[tok] / c[-1] * (2.0 ** -24 + 2.0 ** -38 + off / c[-1])).all()


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_the_lowest_uniform_takes_the_first_kept_element_however_light(rows):
    """u = 0 draws the kept element of the lowest index, also where its weight is far below 2^-52 of the
    row's: a few candidates, a list of them, a cut among many and no filter at all."""
    import torch
    few = np.full(3000, -50.0)
    few[3], few[50] = -4.5, 0.0
    listed = np.full(3000, -60.0)
    listed[500:1499], listed[2500] = -40.0 - np.arange(999) % 7 * 0.125, 0.0
    many = np.full(40960, -80.0)
    many[7], many[2048:22047], many[30000] = -45.5, -44.0 - np.arange(19999) % 5 * 0.25, 0.0
    plain = np.full(40960, -np.inf)
    plain[9], plain[30000:] = -60.0, 0.0
    for x, p, token in ((few, (0.1, 2, 1.0, 0.0), 3), (few, (0.1, 0, 1.0, 1e-20), 3), (listed, (1.0, 1000, 1.0, 0.0), 500),
                        (listed, (1.0, 0, 1.0, 1e-20), 500), (many, (1.0, 20001, 1.0, 0.0), 7), (plain, (1.0, 0, 1.0, 0.0), 9)):
        params, u = records(rows, [p]), np.zeros(rows, np.float32)
        got = run(torch.from_numpy(x[None]).float().cuda(), params, u, ld=0)
        check(got, [x] * rows, params, u, token)
        assert (got[0] == token).all()


@pytest.mark.parametrize("rows", [2, 200])
def test_a_cut_among_masses_below_the_histograms_unit(rows):
    """One heavy element, and 40,959 of some 500 close values that weigh 2^-22 of it together, under the largest
    top_p below 1: its cut lies among masses that no histogram resolves (Z is good to 2^-20 there), so that the
    bracket is halved by exact sums until it fits the list."""
    import torch
    rng = np.random.default_rng([16, rows])
    n = 40960
    x = (-np.log(40959 * 2.0 ** 22) + rng.uniform(-5e-4, 5e-4, n)).astype(np.float32)
    x[1234] = 0.0
    assert 300 < len(np.unique(x)) < 1000
    filters = [(1.0, 0, 1 - 2.0 ** -24, 0.0), (1.0, 30000, 1 - 2.0 ** -24, 0.0), (1.0, 0, 1 - 2.0 ** -23, 0.0)]
    params, u = records(rows, filters), rng.random(rows, np.float32)
    u[:2] = 0.0, 1 - 2.0 ** -24
    got = run(torch.from_numpy(x[None]).cuda(), params, u, ld=0)
    check(got, [x.astype(np.float64)] * rows, params, u)


@pytest.mark.parametrize("n", [4097, 8000, 32003, 65000, 200000, 400001])
def test_lists_as_long_as_they_may_be(n):
    """Cuts at and around what a guessed list holds at each length (fill), up to the list's end and past it, in rows
    of random and of sorted order (where a guess made from the chunks' maxima is wrong) and with closed elements."""
    import torch
    rng = np.random.default_rng([17, n])
    fill = {4097: 72, 8000: 162, 32003: 714, 65000: 1505, 200000: 3696, 400001: 3101}[n]
    x = rng.standard_normal((12, n)) * 3
    x[1::4] = np.sort(x[1::4])[:, ::-1]
    x[2::4][rng.random((3, n)) < 0.5] = -np.inf
    x[3::4, ::128] = np.sort(x[3::4, ::128]) + 9.0  # (every chunk's maximum far above its other elements)
    x = x.astype(np.float32)
    t, want = torch.from_numpy(x).cuda(), x.astype(np.float64)
    reach = np.cumsum(np.sort(np.exp(want[0] - want[0].max()))[::-1])
    mass = [float(reach[c - 1] / reach[-1]) for c in (fill // 2, fill - 1, fill + 1, min(n - 1, 3900))]  # (nuclei of so many)
    filters = [(1.0, k, 1.0, 0.0) for k in (fill - 1, fill, fill + 1, min(4096, n), min(4097, n))]
    filters += [(1.0, 0, p, 0.0) for p in mass] + [(1.0, fill, mass[2], 0.0), (1.0, fill + 50, mass[1], 1e-9)]
    for shift in range(len(filters)):
        params, u = records(12, filters[shift:] + filters[:shift]), rng.random(12, np.float32)
        check(run(t, params, u), want, params, u, shift)
